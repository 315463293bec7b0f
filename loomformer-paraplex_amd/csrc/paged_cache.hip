// Bookkeeping of a paged key-value cache, on the device: forking and freeing
// rows, making the next tokens writable (copy on write), loading dense rows,
// compacting the pool.
//
// A pool has n_pages pages; refs[p] counts the table entries that hold page p
// (0: free).  Row r holds lens[r] tokens (-1: no sequence); its table entries
// below ceil(lens[r] / PS) are its pages, entries behind them are -1, pages
// reserved ahead, which only this row holds, or, where the caller lowered lens[r],
// pages that others may hold too.
#include "loom_common.h"

namespace loom {

constexpr int kPcMaxRows = 1024;
constexpr int kForkCols = 8;        // table columns of a fork block
constexpr int kForkOne = 8192;      // table entries that the reserving block forks itself

struct PageCopy {                   // one copy on write: the first `tokens` tokens of a page
    int32_t src, dst, tokens, pad;
};

struct PoolArgs {
    char* k;
    char* v;
    int64_t layer, page, tok, head;     // strides in bytes
    int layers, KVH, row_bytes;         // row_bytes: HD elements
};

__device__ __forceinline__ bool in_range(int v, int n) { return (unsigned)v < (unsigned)n; }

// ------------------------------------------------------------------ fork

// Row r takes the pages of row parent[r] (none where parent[r] is no row).  A
// block owns kForkCols columns of the whole table: it reads them for all rows,
// then writes, so the gather is in place.  refs change by atomic additions of
// integers: their order does not matter.  256 rows of 67 pages: 3.3 us, bound by
// the latency of a load, an atomic and a store behind the launch.

// The entry that replaces `was` = old[r][c]: the parent's, up to its `held` pages
__device__ __forceinline__ void fork_entry(int32_t* entry, int was, int now, int32_t* refs, int NP) {
    if (was == now) return;
    if (in_range(was, NP)) atomicSub(refs + was, 1);
    if (in_range(now, NP)) atomicAdd(refs + now, 1);
    *entry = now;
}

// Pages of a parent's tokens, those written since (advance) included
__device__ __forceinline__ int held_pages(int len, int advance, int log_ps) {
    return len >= 0 ? (len + advance + (1 << log_ps) - 1) >> log_ps : 0;
}

__global__ void __launch_bounds__(1024)
paged_fork_kernel(int32_t* __restrict__ table, int64_t ld, int MP, const int32_t* __restrict__ lens,
                  int32_t* __restrict__ refs, int NP, int log_ps, const int32_t* __restrict__ parent, int R,
                  int advance) {
    extern __shared__ int32_t old[];                 // [R][kForkCols]
    __shared__ int32_t par[kPcMaxRows], held[kPcMaxRows];
    const int c0 = blockIdx.x * kForkCols, tid = threadIdx.x;
    for (int i = tid; i < R * kForkCols; i += 1024) {
        const int c = c0 + i % kForkCols;
        old[i] = c < MP ? table[(int64_t)(i / kForkCols) * ld + c] : -1;
    }
    if (tid < R) {
        const int p = parent[tid];
        par[tid] = p;
        held[tid] = in_range(p, R) ? held_pages(lens[p], advance, log_ps) : 0;
    }
    __syncthreads();
    for (int i = tid; i < R * kForkCols; i += 1024) {
        const int r = i / kForkCols, cc = i % kForkCols, c = c0 + cc, p = par[r];
        if (c >= MP || p == r) continue;
        fork_entry(table + (int64_t)r * ld + c, old[i], c < held[r] ? old[p * kForkCols + cc] : -1, refs, NP);
    }
}

// ------------------------------------------------------------------ reserve

// Exclusive scan of N counts over the 1024 threads of a block; total: their sums.
template <int N>
__device__ __forceinline__ void block_scan(const int (&v)[N], int (*waves)[N], int (&before)[N], int (&total)[N]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int incl[N];
    __syncthreads();                                 // the previous use of `waves` is over
#pragma unroll
    for (int k = 0; k < N; ++k) {
        incl[k] = wave_scan_int(v[k]);
        if (lane == 63) waves[wave][k] = incl[k];
    }
    __syncthreads();
    // lane w of every wave holds wave w's sums
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int mine = lane < 16 ? waves[lane][k] : 0;
        const int upto = wave_scan_int(mine);
        total[k] = __builtin_amdgcn_readlane(upto, 15);
        before[k] = __builtin_amdgcn_readlane(upto - mine, __builtin_amdgcn_readfirstlane(wave)) + incl[k] - v[k];
    }
}

constexpr int kScanIds = 4;         // groups of four page ids per thread and round

// One block.  lens[r] = lens[parent[r]] + advance, then the tokens lens[r] ..
// lens[r] + n_new - 1 (n_new: n_each[r], or n_all for every row) get pages of their own: where the row's last page is
// partly filled and held more than once, row order decides who copies it (each
// row in turn copies while others hold it), and pages that are missing are
// appended.  A row lets go of pages in their places that others hold too (they hold
// none of its tokens), and of what lies behind the first of them.  The free pages are taken lowest id first, in row order, by one
// scan over refs: a free page's rank among the free ones names its row.
// Bound by the latency of its stages, each a pass over the rows or over refs with a
// block scan behind it: 256 rows, 67 places each, 8.8 us; 64 rows that get up to 128 pages each
// 11.6, one row that gets 1024 38 (its thread walks its places).  One block and not a launch
// per stage, since each stage needs the whole of the one before.
// FORK: the block also forks the table, staged whole in LDS: a launch less, but
// one CU's work.  All of a call in both forms (us, one launch / two): 92 entries
// 8.0 / 9.9, 4384 10.6 / 11.1, 17152 20.5 / 17.2, 32512 19.6 / 13.7.
template <bool FORK>
__global__ void __launch_bounds__(1024)
paged_reserve_kernel(int32_t* __restrict__ table, int64_t ld, int MP, int32_t* __restrict__ lens,
                     int32_t* refs, int NP, int log_ps, const int32_t* __restrict__ parent, int R,
                     int n_all, const int32_t* __restrict__ n_each, int advance, PageCopy* __restrict__ copies,
                     int32_t* __restrict__ status) {
    extern __shared__ int32_t old[];                 // FORK: [R][MP]
    __shared__ __align__(16) int32_t tail[kPcMaxRows];
    __shared__ int32_t base[kPcMaxRows], slot0[kPcMaxRows], len_of[kPcMaxRows];
    __shared__ int waves[16][2], ahead;              // ahead: a row has a page behind its tokens
    const int r = threadIdx.x, PS = 1 << log_ps;
    // a page's count where this block may have changed it since it was last read
    auto count_of = [&](int64_t id) __attribute__((always_inline)) {
        return __hip_atomic_load(refs + id, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
    // bit 4 j + e: page seg + 4096 j + 4 r + e is free
    auto free_ids = [&](int64_t seg, bool changed) __attribute__((always_inline)) {
        uint32_t mask = 0;
#pragma unroll
        for (int j = 0; j < kScanIds; ++j) {
            const int64_t id = seg + 4096 * j + 4 * r;
            if (changed) {
                for (int e = 0; e < 4 && id + e < NP; ++e)
                    if (count_of(id + e) <= 0) mask |= 1u << (4 * j + e);
            } else if (id + 4 <= NP) {
                int4 q;                              // one load, aligned to a word
                __builtin_memcpy(&q, refs + id, 16);
                mask |= (uint32_t)((q.x <= 0) | (q.y <= 0) << 1 | (q.z <= 0) << 2 | (q.w <= 0) << 3) << (4 * j);
            } else {
                for (int e = 0; e < 4 && id + e < NP; ++e)
                    if (refs[id + e] <= 0) mask |= 1u << (4 * j + e);
            }
        }
        return mask;
    };
    uint32_t mask = 0;                               // of the first pages, with the row's first loads
    if constexpr (!FORK) mask = free_ids(0, false);
    if (r == 0) ahead = 0;
    // (r + 1024 k) as (row, column), without a division per entry
    const int step_r = 1024 / MP, step_c = 1024 - step_r * MP;
    int len = -1, p = -1;
    if (r < R) p = parent != nullptr ? parent[r] : r;
    if constexpr (FORK) {
        constexpr int kU = 8;                        // loads in flight
        int er = r / MP, ec = r - er * MP;
        for (int i0 = r; i0 < R * MP; i0 += 1024 * kU) {
            int32_t v[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                v[u] = i0 + 1024 * u < R * MP ? table[(int64_t)er * ld + ec] : -1;
                er += step_r;
                ec += step_c;
                if (ec >= MP) {
                    ec -= MP;
                    ++er;
                }
            }
#pragma unroll
            for (int u = 0; u < kU; ++u)
                if (i0 + 1024 * u < R * MP) old[i0 + 1024 * u] = v[u];
        }
    }
    if (in_range(p, R)) len = lens[p];
    len = len >= 0 ? len + advance : -1;
    // base: the row's parent, slot0: the pages it takes from it (both until the scan)
    base[r] = p;
    slot0[r] = held_pages(len, 0, log_ps);
    len_of[r] = len;
    __syncthreads();                                 // every parent's length is read
    if (r < R && n_each == nullptr) lens[r] = len;   // (a reservation per row leaves lens alone)
    if constexpr (FORK) {
        int er = r / MP, ec = r - er * MP;
        for (int i = r; i < R * MP; i += 1024) {
            const int q = base[er];
            if (q != er) fork_entry(table + (int64_t)er * ld + ec, old[i], ec < slot0[er] ? old[q * MP + ec] : -1, refs, NP);
            er += step_r;
            ec += step_c;
            if (ec >= MP) {
                ec -= MP;
                ++er;
            }
        }
    }
    int32_t* row = table + (int64_t)r * ld;
    const int held = slot0[r];
    // the row's entry as it is now
    auto entry = [&](int s) __attribute__((always_inline)) {
        if constexpr (FORK) return p == r ? old[r * MP + s] : s < held ? old[p * MP + s] : -1;
        else return row[s];
    };
    int page = -1, short_of = 0;
    bool copy = false;
    const int cap = MP * PS;
    const int n_new = n_each != nullptr ? (r < R ? max(n_each[r], 0) : 0) : n_all;
    const int n = len >= 0 ? max(min(n_new, cap - len), 0) : 0;
    if (len >= 0 && n < n_new) short_of = 1;
    int miss0 = 0, last = -1;
    if (n > 0) {
        if (len & (PS - 1)) {
            page = entry(len >> log_ps);
            if (!in_range(page, NP)) page = -1;
        }
        last = (len + n - 1) >> log_ps;
        miss0 = (len + PS - 1) >> log_ps;
        bool any = false;
#pragma unroll 4
        for (int s = miss0; s <= last; ++s) any |= in_range(entry(s), NP);
        if (any) ahead = 1;
    }
    tail[r] = page;
    __syncthreads();                                 // (and the fork's changes of refs are done)
    const bool let_go = ahead != 0;
    if (let_go) {                                    // (the same in all threads)
        while (miss0 <= last && in_range(entry(miss0), NP) && count_of(entry(miss0)) <= 1) ++miss0;
        __syncthreads();                             // every row goes by the counts as they were
        for (int s = miss0; s <= last; ++s) {
            const int e = entry(s);
            if (!in_range(e, NP)) continue;
            row[s] = -1;
            atomicSub(refs + e, 1);
        }
        __syncthreads();
        if constexpr (!FORK) mask = free_ids(0, true);
    }
    const int nmiss = last + 1 - miss0;
    const int held_by = page >= 0 ? count_of(page) : 0;
    // rows before this one with the same tail: `share` threads count for a row
    int share = 16;
    while (share > 1 && R * share > 1024) share >>= 1;
    const int of = r / share, part = r & (share - 1);
    if (of < R) {
        const int mine = tail[of];
        int before = 0;
        if (mine >= 0) {
#pragma unroll 4
            for (int i = 4 * part; i < of; i += 4 * share) {
                const int4 t = *reinterpret_cast<const int4*>(tail + i);
                before += (t.x == mine) + (i + 1 < of && t.y == mine) + (i + 2 < of && t.z == mine) +
                          (i + 3 < of && t.w == mine);
            }
        }
        if (share >= 2) before += __builtin_amdgcn_update_dpp(0, before, kDppQuad1032, 0xF, 0xF, false);
        if (share >= 4) before += __builtin_amdgcn_update_dpp(0, before, kDppQuad2301, 0xF, 0xF, false);
        if (share >= 8) before += __builtin_amdgcn_update_dpp(0, before, kDppHalfMirror, 0xF, 0xF, false);
        if (share >= 16) before += __builtin_amdgcn_update_dpp(0, before, kDppMirror, 0xF, 0xF, false);
        if (part == 0) base[of] = before;
    }
    __syncthreads();
    copy = page >= 0 && held_by - base[r] > 1;
    const int want = nmiss + (copy ? 1 : 0);
    int want1[1] = {want}, first1[1], total1[1];
    block_scan<1>(want1, reinterpret_cast<int(*)[1]>(waves), first1, total1);
    const int first = first1[0];
    base[r] = first;
    slot0[r] = copy ? ~miss0 : miss0;                // (the sign says whether the first page is a copy's)
    if (r < R) copies[r] = PageCopy{-1, -1, 0, 0};
    const int need = total1[0];
    int given = 0;                                   // free pages handed out so far
    __syncthreads();
    for (int64_t seg = 0; seg < NP && given < need; seg += 1024 * 4 * kScanIds) {
        if (FORK || seg > 0) mask = free_ids(seg, let_go);
        int count[2] = {0, 0}, before[2], all[2];    // 16 bits per j
#pragma unroll
        for (int j = 0; j < kScanIds; ++j) count[j / 2] |= __popc((mask >> (4 * j)) & 15u) << (16 * (j & 1));
        block_scan<2>(count, waves, before, all);
#pragma unroll
        for (int j = 0; j < kScanIds; ++j) {
            const uint32_t bits = (mask >> (4 * j)) & 15u;
            int rank = given + ((before[j / 2] >> (16 * (j & 1))) & 0xffff);
            if (bits != 0 && rank < need) {
                int lo = 0, hi = R - 1;              // the last row whose base is at most `rank`
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (base[mid] <= rank) lo = mid; else hi = mid - 1;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (!((bits >> e) & 1u) || rank >= need) continue;
                    while (lo + 1 < R && base[lo + 1] <= rank) ++lo;
                    const int id = (int)(seg + 4096 * j + 4 * r + e);
                    const bool cp = slot0[lo] < 0;
                    const int k = rank - base[lo], m0 = cp ? ~slot0[lo] : slot0[lo];
                    refs[id] = 1;
                    if (cp && k == 0) {
                        const int l = len_of[lo], sl = l >> log_ps;
                        copies[lo] = PageCopy{tail[lo], id, l & (PS - 1), 0};
                        table[(int64_t)lo * ld + sl] = id;
                        atomicSub(refs + tail[lo], 1);
                    } else {
                        table[(int64_t)lo * ld + m0 + k - (cp ? 1 : 0)] = id;
                    }
                    ++rank;
                }
            }
            given += (all[j / 2] >> (16 * (j & 1))) & 0xffff;
        }
    }
    // a row whose copy found no page must not write into the shared one
    if (copy && first >= given) {
        row[len >> log_ps] = -1;
        atomicSub(refs + page, 1);
    }
    if (short_of) atomicAdd(status, 1);
    if (r == 0 && given < need) atomicAdd(status, need - given);
}

// Copies of `copies[r]`, both pools of all layers: block (r, y) takes every
// gridDim.y-th of the row's 2 * layers pages, as one run of pieces, kCowUnroll in
// flight per thread.  Bound by the copy of what the rows share: 4 rows that
// share 13 tokens of 10 layers, 2 kv heads of 96, 2.9 us, most of it the launch; 256
// rows that share 4 tokens 4.7 us.
constexpr int kCowUnroll = 4;

__global__ void __launch_bounds__(256)
paged_cow_kernel(PoolArgs a, const PageCopy* __restrict__ copies) {
    const PageCopy c = copies[blockIdx.x];
    if (c.src < 0) return;
    const uint32_t pieces = a.row_bytes / 16, per_head = c.tokens * pieces, per_page = a.KVH * per_head;
    const uint32_t pages = (2 * a.layers - blockIdx.y + gridDim.y - 1) / gridDim.y;
    for (uint32_t i0 = threadIdx.x; i0 < pages * per_page; i0 += 256 * kCowUnroll) {
        u32x4 v[kCowUnroll];
        char* to[kCowUnroll];
#pragma unroll
        for (int u = 0; u < kCowUnroll; ++u) {
            const uint32_t i = i0 + 256 * u;
            if (i >= pages * per_page) continue;
            const uint32_t n = i / per_page, k = i - n * per_page, h = k / per_head, m = k - h * per_head, t = m / pieces;
            const uint32_t lp = blockIdx.y + n * gridDim.y;
            char* pool = (lp & 1 ? a.v : a.k) + (int64_t)(lp >> 1) * a.layer + h * a.head + t * a.tok +
                         (int64_t)(m - t * pieces) * 16;
            to[u] = pool + c.dst * a.page;
            v[u] = *reinterpret_cast<const u32x4*>(pool + c.src * a.page);
        }
#pragma unroll
        for (int u = 0; u < kCowUnroll; ++u)
            if (i0 + 256 * u < pages * per_page) *reinterpret_cast<u32x4*>(to[u]) = v[u];
    }
}

// ------------------------------------------------------------------ dense rows into pages

// Tokens first[r] .. last[r] - 1 of row r of a dense cache (element (layer, r,
// head, t) at the strides given) into the row's pages: grid (token tiles of
// kWriteTile, rows, layers * KVH * 2).  Tokens without a page are left out.  A copy:
// each 16 bytes are read once and written once, a run of a head's tokens per block.
// 32 rows of 2048 tokens, 10 layers, 2 kv heads of 96, bf16, 1.0 GB read and written:
// 183 us, 5.5 TB/s; one row of 512, 4.8 us.
constexpr int kWriteTile = 64;

__global__ void __launch_bounds__(256)
paged_write_kernel(PoolArgs a, const char* __restrict__ kd, const char* __restrict__ vd, int64_t s_layer,
                   int64_t s_row, int64_t s_head, int64_t s_tok, int T, const int32_t* __restrict__ table,
                   int64_t ld, int MP, int NP, int log_ps, const int32_t* __restrict__ first,
                   const int32_t* __restrict__ last) {
    const int r = blockIdx.y, t0 = blockIdx.x * kWriteTile;
    const int lo = max(max(first[r], 0), t0);
    const int hi = min(min(min(last[r], T), MP << log_ps), t0 + kWriteTile);
    if (lo >= hi) return;
    const int z = blockIdx.z, which = z & 1, h = (z >> 1) % a.KVH;
    const int64_t l = (z >> 1) / a.KVH;
    char* pool = (which ? a.v : a.k) + l * a.layer + h * a.head;
    const char* src = (which ? vd : kd) + l * s_layer + r * s_row + h * s_head;
    const int pieces = a.row_bytes / 16, mask = (1 << log_ps) - 1;
    for (int i = threadIdx.x; i < (hi - lo) * pieces; i += 256) {
        const int t = lo + i / pieces, c = i % pieces;
        const int page = table[(int64_t)r * ld + (t >> log_ps)];
        if (!in_range(page, NP)) continue;
        *reinterpret_cast<u32x4*>(pool + page * a.page + (int64_t)(t & mask) * a.tok + 16 * c) =
            *reinterpret_cast<const u32x4*>(src + (int64_t)t * s_tok + 16 * c);
    }
}

// ------------------------------------------------------------------ compact

// One block: U = pages in use; the k-th used page with id >= U (movers) goes to
// the k-th free id below U (holes); map[p] = the new id of page p.  ws: [0] the
// number of moves, then movers [NP], holes [NP], map [NP].  Two block scans over
// refs: 6000 pages 7.7 us, 151 pages 2.8 us.
__global__ void __launch_bounds__(1024)
paged_compact_plan_kernel(int32_t* refs, int NP, int32_t* __restrict__ used, int32_t* ws) {
    __shared__ int waves[16][2];
    int32_t *movers = ws + 4, *holes = movers + NP, *map = holes + NP;
    const int r = threadIdx.x;
    int mine[1] = {0}, ignore[1], total[1];
    for (int64_t i = r; i < NP; i += 1024) mine[0] += refs[i] > 0;
    block_scan<1>(mine, reinterpret_cast<int(*)[1]>(waves), ignore, total);
    const int U = total[0];
    int nm = 0, nh = 0;
    for (int64_t seg = 0; seg < NP; seg += 4096) {
        int count[2] = {0, 0}, before[2], all[2];    // movers, holes
        uint32_t bits = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t id = seg + 4 * r + e;
            if (id >= NP) continue;
            const bool inuse = refs[id] > 0;
            map[id] = (int)id;
            if (inuse && id >= U) { ++count[0]; bits |= 1u << e; }
            if (!inuse && id < U) { ++count[1]; bits |= 16u << e; }
        }
        block_scan<2>(count, waves, before, all);
        int m = nm + before[0], h = nh + before[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int id = (int)(seg + 4 * r + e);
            if (bits >> e & 1u) movers[m++] = id;
            if (bits >> (4 + e) & 1u) holes[h++] = id;
        }
        nm += all[0];
        nh += all[1];
    }
    __syncthreads();                                 // the lists and the map are written
    for (int i = r; i < nm; i += 1024) {             // (as many holes as movers)
        const int from = movers[i], to = holes[i];
        map[from] = to;
        refs[to] = refs[from];
        refs[from] = 0;
    }
    if (r == 0) {
        ws[0] = nm;
        *used = U;
    }
}

constexpr int kMoveUnroll = 6;      // 16-byte pieces in flight per thread

// The moves (a page of one layer's K or V pool each) and, in the blocks of
// y = 1, the tables' new ids.  Bound by the copy, read and written once: 6000 pages
// of 64 tokens, 10 layers, 2 kv heads of 96, bf16, a third of them in use, 1.31 GB read
// and written: 257 us, 5.1 TB/s (a large copy: 5.2).  2, 6 or 8 pieces in flight: 269, 271, 269 us with the plan.
__global__ void __launch_bounds__(256)
paged_compact_move_kernel(PoolArgs a, int PS, const int32_t* __restrict__ ws, int NP, int32_t* __restrict__ table,
                          int64_t ld, int MP, int R) {
    const int32_t *movers = ws + 4, *holes = movers + NP, *map = holes + NP;
    if (blockIdx.y == 1) {
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)R * MP; i += (int64_t)gridDim.x * 256) {
            int32_t* e = table + (i / MP) * ld + i % MP;
            const int p = *e;
            if (in_range(p, NP)) *e = map[p];
        }
        return;
    }
    // a page as runs of bytes that lie together: the whole page where heads and
    // tokens follow each other, else a head's tokens, else a token
    const int64_t units = (int64_t)ws[0] * 2 * a.layers;
    const bool head_run = a.tok == a.row_bytes, page_run = head_run && a.head == (int64_t)PS * a.row_bytes;
    const int runs = page_run ? 1 : head_run ? a.KVH : a.KVH * PS;
    // (a page may have almost 2^31 bytes, so places in it plus a step need the 32nd bit)
    const uint32_t run = page_run ? a.KVH * PS * a.row_bytes : head_run ? PS * a.row_bytes : a.row_bytes;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int i = (int)(u / (2 * a.layers)), lp = (int)(u - (int64_t)i * 2 * a.layers);
        char* pool = (lp & 1 ? a.v : a.k) + (int64_t)(lp >> 1) * a.layer;
        const char* src = pool + movers[i] * a.page;
        char* dst = pool + holes[i] * a.page;
        for (int n = 0; n < runs; ++n) {
            const int64_t off = page_run ? 0 : head_run ? n * a.head : (n / PS) * a.head + (n % PS) * a.tok;
            for (uint32_t b0 = threadIdx.x * 16; b0 < run; b0 += 256 * 16 * kMoveUnroll) {
                u32x4 v[kMoveUnroll];
#pragma unroll
                for (int k = 0; k < kMoveUnroll; ++k)
                    if (b0 + 4096 * k < run)
                        v[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + off + b0 + 4096 * k));
#pragma unroll
                for (int k = 0; k < kMoveUnroll; ++k)
                    if (b0 + 4096 * k < run)
                        __builtin_nontemporal_store(v[k], reinterpret_cast<u32x4*>(dst + off + b0 + 4096 * k));
            }
        }
    }
}

// ------------------------------------------------------------------ host side

static int pool_checks(const char* who, int dtype, const void* k, const void* v, int64_t L, int64_t layer,
                       int64_t page, int64_t tok, int64_t head, int64_t NP, int64_t PS, int64_t KVH, int64_t HD,
                       PoolArgs* out) {
    LOOM_CHECK(dtype == LOOM_F32 || dtype == LOOM_BF16 || dtype == LOOM_F16, "%s: unsupported dtype %d", who, dtype);
    const int64_t es = dtype == LOOM_F32 ? 4 : 2;
    LOOM_CHECK(PS >= 16 && PS <= 1024 && (PS & (PS - 1)) == 0,
               "%s: page_size must be a power of two from 16 to 1024, got %lld", who, (long long)PS);
    LOOM_CHECK(NP >= 1 && NP < ((int64_t)1 << 30), "%s: bad n_pages %lld", who, (long long)NP);
    LOOM_CHECK(L >= 1 && L <= 4096 && KVH >= 1 && KVH <= 4096 && HD >= 8 && HD <= 1024 && HD % 8 == 0,
               "%s: bad pool shape layers=%lld heads=%lld head_dim=%lld", who, (long long)L, (long long)KVH, (long long)HD);
    LOOM_CHECK(tok >= HD && page >= 0 && head >= 0 && layer >= 0, "%s: bad pool strides", who);
    LOOM_CHECK((tok * es) % 16 == 0 && (page * es) % 16 == 0 && (head * es) % 16 == 0 && (layer * es) % 16 == 0 &&
                   k != nullptr && v != nullptr && (((uintptr_t)k | (uintptr_t)v) % 16) == 0,
               "%s: the pools must be given, they and their strides multiples of 16 bytes", who);
    LOOM_CHECK(KVH * PS * HD * es < ((int64_t)1 << 31) && 2 * L * KVH * PS * HD * es / 16 < ((int64_t)1 << 31),
               "%s: a page of %lld bytes in %lld layers is more than a copy takes at once", who,
               (long long)(KVH * PS * HD * es), (long long)L);
    *out = PoolArgs{(char*)k, (char*)v, layer * es, page * es, tok * es, head * es, (int)L, (int)KVH, (int)(HD * es)};
    return LOOM_OK;
}

static int table_checks(const char* who, const int32_t* table, int64_t ld, int64_t MP, int64_t PS, int64_t R) {
    LOOM_CHECK(R >= 0 && R <= kPcMaxRows, "%s: 0 to %d rows, got %lld", who, kPcMaxRows, (long long)R);
    LOOM_CHECK(MP >= 1 && MP <= ((int64_t)1 << 24) / PS && ld >= MP,
               "%s: the table must hold 1 page to 2^24 tokens per row (max_pages=%lld, row stride %lld)", who,
               (long long)MP, (long long)ld);
    LOOM_CHECK(table != nullptr || R == 0, "%s: a required pointer is NULL", who);
    return LOOM_OK;
}

// The copies that a reservation listed
static int cow_launch(const char* who, const PoolArgs& a, int64_t rows, const void* copies, hipStream_t st) {
    // (about 2048 blocks, and no more than a block per page)
    const int64_t y = ceil_div((int64_t)2048, rows), pages = 2 * (int64_t)a.layers;
    hipLaunchKernelGGL(paged_cow_kernel, dim3((unsigned)rows, (unsigned)(y < pages ? y : pages)), dim3(256), 0, st, a,
                       (const PageCopy*)copies);
    return launch_status(who);
}

}  // namespace loom

using namespace loom;

extern "C" int64_t loom_paged_update_workspace_bytes(int64_t rows) {
    return rows > 0 ? rows * (int64_t)sizeof(PageCopy) : 0;
}

extern "C" int loom_paged_update(int dtype, void* k_pages, void* v_pages, int64_t layers, int64_t layer_stride,
                                 int64_t page_stride, int64_t token_stride, int64_t head_stride, int64_t n_pages,
                                 int64_t page_size, int64_t KVH, int64_t HD, int32_t* table, int64_t table_ld,
                                 int64_t max_pages, int32_t* lens, int32_t* refs, int32_t* status,
                                 const int32_t* parent, int64_t n_new, int64_t advance, void* workspace,
                                 int64_t workspace_bytes, int64_t rows, void* stream) {
    clear_error();
    const char* who = "paged_update";
    PoolArgs a;
    if (int rc = pool_checks(who, dtype, k_pages, v_pages, layers, layer_stride, page_stride, token_stride,
                             head_stride, n_pages, page_size, KVH, HD, &a))
        return rc;
    if (int rc = table_checks(who, table, table_ld, max_pages, page_size, rows)) return rc;
    LOOM_CHECK((lens && refs && status) || rows == 0, "%s: a required pointer is NULL", who);
    LOOM_CHECK(n_new >= 0 && n_new <= max_pages * page_size && advance >= 0 && advance <= max_pages * page_size,
               "%s: n_new=%lld and advance=%lld must lie in 0..%lld", who, (long long)n_new, (long long)advance,
               (long long)(max_pages * page_size));
    LOOM_CHECK(workspace_bytes >= loom_paged_update_workspace_bytes(rows) && (workspace != nullptr || rows == 0) &&
                   ((uintptr_t)workspace % 16) == 0,
               "%s: a 16-byte aligned workspace of %lld bytes is needed, got %lld", who,
               (long long)loom_paged_update_workspace_bytes(rows), (long long)workspace_bytes);
    if (rows == 0) return LOOM_OK;
    hipStream_t st = (hipStream_t)stream;
    const int log_ps = __builtin_ctzll((unsigned long long)page_size);
    const bool fork = parent != nullptr, one = fork && rows * max_pages <= kForkOne;
    if (fork && !one) {
        hipLaunchKernelGGL(paged_fork_kernel, dim3((unsigned)ceil_div(max_pages, kForkCols)), dim3(1024),
                           (unsigned)(rows * kForkCols * sizeof(int32_t)), st, table, table_ld, (int)max_pages, lens,
                           refs, (int)n_pages, log_ps, parent, (int)rows, (int)advance);
        if (int rc = launch_status("loom_paged_update(fork)")) return rc;
    }
    if (!fork && n_new == 0 && advance == 0) return LOOM_OK;
    if (one)
        hipLaunchKernelGGL((paged_reserve_kernel<true>), dim3(1), dim3(1024), (unsigned)(rows * max_pages * sizeof(int32_t)),
                           st, table, table_ld, (int)max_pages, lens, refs, (int)n_pages, log_ps, parent, (int)rows,
                           (int)n_new, (const int32_t*)nullptr, (int)advance, (PageCopy*)workspace, status);
    else
        hipLaunchKernelGGL((paged_reserve_kernel<false>), dim3(1), dim3(1024), 0, st, table, table_ld, (int)max_pages,
                           lens, refs, (int)n_pages, log_ps, parent, (int)rows, (int)n_new, (const int32_t*)nullptr, (int)advance,
                           (PageCopy*)workspace, status);
    if (int rc = launch_status("loom_paged_update(reserve)")) return rc;
    if (n_new == 0) return LOOM_OK;
    return cow_launch("loom_paged_update(copy)", a, rows, workspace, st);
}

extern "C" int loom_paged_reserve(int dtype, void* k_pages, void* v_pages, int64_t layers, int64_t layer_stride,
                                  int64_t page_stride, int64_t token_stride, int64_t head_stride, int64_t n_pages,
                                  int64_t page_size, int64_t KVH, int64_t HD, int32_t* table, int64_t table_ld,
                                  int64_t max_pages, int32_t* lens, int32_t* refs, int32_t* status,
                                  const int32_t* new_tokens, void* workspace, int64_t workspace_bytes, int64_t rows,
                                  void* stream) {
    clear_error();
    const char* who = "paged_reserve";
    PoolArgs a;
    if (int rc = pool_checks(who, dtype, k_pages, v_pages, layers, layer_stride, page_stride, token_stride,
                             head_stride, n_pages, page_size, KVH, HD, &a))
        return rc;
    if (int rc = table_checks(who, table, table_ld, max_pages, page_size, rows)) return rc;
    LOOM_CHECK((lens && refs && status && new_tokens) || rows == 0, "%s: a required pointer is NULL", who);
    LOOM_CHECK(workspace_bytes >= loom_paged_update_workspace_bytes(rows) && (workspace != nullptr || rows == 0) &&
                   ((uintptr_t)workspace % 16) == 0,
               "%s: a 16-byte aligned workspace of %lld bytes is needed, got %lld", who,
               (long long)loom_paged_update_workspace_bytes(rows), (long long)workspace_bytes);
    if (rows == 0) return LOOM_OK;
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL((paged_reserve_kernel<false>), dim3(1), dim3(1024), 0, st, table, table_ld, (int)max_pages,
                       lens, refs, (int)n_pages, __builtin_ctzll((unsigned long long)page_size), (const int32_t*)nullptr,
                       (int)rows, 0, new_tokens, 0, (PageCopy*)workspace, status);
    if (int rc = launch_status("loom_paged_reserve(reserve)")) return rc;
    return cow_launch("loom_paged_reserve(copy)", a, rows, workspace, st);
}

extern "C" int loom_paged_write(int dtype, void* k_pages, void* v_pages, int64_t layers, int64_t layer_stride,
                                int64_t page_stride, int64_t token_stride, int64_t head_stride, int64_t n_pages,
                                int64_t page_size, int64_t KVH, int64_t HD, const int32_t* table, int64_t table_ld,
                                int64_t max_pages, const void* k_rows, const void* v_rows, int64_t src_layer_stride,
                                int64_t src_row_stride, int64_t src_head_stride, int64_t src_token_stride,
                                int64_t src_tokens, const int32_t* first, const int32_t* last, int64_t rows,
                                void* stream) {
    clear_error();
    const char* who = "paged_write";
    PoolArgs a;
    if (int rc = pool_checks(who, dtype, k_pages, v_pages, layers, layer_stride, page_stride, token_stride,
                             head_stride, n_pages, page_size, KVH, HD, &a))
        return rc;
    if (int rc = table_checks(who, table, table_ld, max_pages, page_size, rows)) return rc;
    const int64_t es = dtype == LOOM_F32 ? 4 : 2;
    LOOM_CHECK((k_rows && v_rows && first && last) || rows == 0, "%s: a required pointer is NULL", who);
    LOOM_CHECK(src_tokens >= 0 && src_tokens <= ((int64_t)1 << 24) && src_token_stride >= HD &&
                   src_layer_stride >= 0 && src_row_stride >= 0 && src_head_stride >= 0,
               "%s: bad source shape", who);
    LOOM_CHECK((src_layer_stride * es) % 16 == 0 && (src_row_stride * es) % 16 == 0 &&
                   (src_head_stride * es) % 16 == 0 && (src_token_stride * es) % 16 == 0 &&
                   (((uintptr_t)k_rows | (uintptr_t)v_rows) % 16) == 0,
               "%s: the source rows and their strides must be multiples of 16 bytes", who);
    LOOM_CHECK(2 * layers * KVH <= 65535, "%s: too many layers x heads", who);
    if (rows == 0 || src_tokens == 0) return LOOM_OK;
    const int64_t tiles = ceil_div(src_tokens, kWriteTile);
    hipLaunchKernelGGL(paged_write_kernel, dim3((unsigned)tiles, (unsigned)rows, (unsigned)(2 * layers * KVH)),
                       dim3(256), 0, (hipStream_t)stream, a, (const char*)k_rows, (const char*)v_rows,
                       src_layer_stride * es, src_row_stride * es, src_head_stride * es, src_token_stride * es,
                       (int)src_tokens, table, table_ld, (int)max_pages, (int)n_pages,
                       __builtin_ctzll((unsigned long long)page_size), first, last);
    return launch_status("loom_paged_write");
}

extern "C" int64_t loom_paged_compact_workspace_bytes(int64_t n_pages) {
    return n_pages > 0 ? (4 + 3 * n_pages) * (int64_t)sizeof(int32_t) : 0;
}

extern "C" int loom_paged_compact(int dtype, void* k_pages, void* v_pages, int64_t layers, int64_t layer_stride,
                                  int64_t page_stride, int64_t token_stride, int64_t head_stride, int64_t n_pages,
                                  int64_t page_size, int64_t KVH, int64_t HD, int32_t* table, int64_t table_ld,
                                  int64_t max_pages, int32_t* refs, int32_t* used, void* workspace,
                                  int64_t workspace_bytes, int64_t rows, void* stream) {
    clear_error();
    const char* who = "paged_compact";
    PoolArgs a;
    if (int rc = pool_checks(who, dtype, k_pages, v_pages, layers, layer_stride, page_stride, token_stride,
                             head_stride, n_pages, page_size, KVH, HD, &a))
        return rc;
    if (int rc = table_checks(who, table, table_ld, max_pages, page_size, rows)) return rc;
    LOOM_CHECK(refs && used, "%s: a required pointer is NULL", who);
    LOOM_CHECK(workspace_bytes >= loom_paged_compact_workspace_bytes(n_pages) && workspace != nullptr &&
                   ((uintptr_t)workspace % 16) == 0,
               "%s: a 16-byte aligned workspace of %lld bytes is needed, got %lld", who,
               (long long)loom_paged_compact_workspace_bytes(n_pages), (long long)workspace_bytes);
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(paged_compact_plan_kernel, dim3(1), dim3(1024), 0, st, refs, (int)n_pages, used,
                       (int32_t*)workspace);
    if (int rc = launch_status("loom_paged_compact(plan)")) return rc;
    hipLaunchKernelGGL(paged_compact_move_kernel, dim3((unsigned)(8 * device_cus()), 2), dim3(256), 0, st, a,
                       (int)page_size, (const int32_t*)workspace, (int)n_pages, table, table_ld, (int)max_pages,
                       (int)rows);
    return launch_status("loom_paged_compact(move)");
}
