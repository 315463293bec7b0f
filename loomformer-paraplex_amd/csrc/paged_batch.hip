// A serving step over a paged key-value cache, for gfx950: every row of the batch
// brings a number of new tokens of its own (none, one, a whole prompt), and pages
// that rows have in common are read once for all of them.
//
// Token t of row r, the i-th of its new ones, stands at position p = lens[r] + i and
// attends to positions 0 .. p of its row.  With s_j = q . k_j / sqrt(HD):
//   C = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  Kctx = the same of k_j.
// The sums split over any partition of the positions: each part leaves (m, l, C, Kctx)
// with its own maximum m and sum l, and the join weighs them by e^(m - max m).  The
// partition is that of the work: the positions that rows share against all those
// rows' queries at once, then each row's own.
//
// What rows share is one run of whole pages per first page: rows of up to kPbAlone queries that begin
// with the same page are a group, and the run is the least that all its rows have in common.  A
// row that parts early cuts it for the others (64 rows behind 16384 of which one parts after
// 64: items 249 us, 52 without it).
//
// Which rows share what only the device knows, so a step is planned there, once for
// all layers:
//   rows     which rows begin with the same pages, and how many (paged_rows_kernel)
//   plan     segments (a block of up to 128 queries and the positions they read), cut
//            into items of about equal work, one block each (paged_plan_kernel)
// and a layer is three launches: rope and append, the items, the join.
#include "attn_tile.h"
#include "paged_math.h"

#include <type_traits>

namespace loom {

constexpr int kPbMaxRows = 1024;
constexpr int kPbQ = 128;           // queries (a token's heads of one kv head) of a block
constexpr int kPbTile = 64;         // positions of a step of a block
constexpr int kPbLeast = 1;         // an item has so many tiles at least
constexpr float kPbRecord = 4e-4f;  // a query's record, in a block's time for a tile of its queries
constexpr int kPbFew = 8;           // records of a query that a wave of the join takes alone
constexpr int kPbAlone = 64;        // rows with more queries fill a block by themselves and share nothing
constexpr int kPbShare = 64;        // common positions from which reading them once pays
constexpr int kPbMagic = 0x4c50424c;
constexpr int64_t kPbMaxTokens = (int64_t)1 << 20;

// A block of queries and the positions they read.  Query x (0 .. nq - 1) is query x0 +
// x of a list of tokens times the kv head's G heads: token list entry (x0 + x) / G,
// head (x0 + x) % G.  An item is a segment's tiles tile0 .. tile1 - 1, the work of a block.
constexpr int kPbOwn = 0, kPbRun = 1, kPbList = 2;   // the list: a row's own tokens, a group's that
                                                     // lie one behind the other, or a group's in toks
struct alignas(64) PbItem {
    int row;                        // whose table entries name the pages
    int key0, key1;                 // positions key0 .. key1 - 1, key0 a multiple of 16
    int base;                       // the list's first token (or its place in toks)
    int x0, nq;
    int lens;                       // own: tokens the row held before the step
    int kind;
    int tile0, tile1;
    int rec;                        // the item's record of query x is rec + x (< 0: none)
    int pad[5];
};

// An own segment whose queries' sums are in records: of query x, records own + x and every
// nq-th behind it, own_n in all, and, where the row shares positions, common_n of the group's segment
// that holds the query, which is the g0 + x-th of the group's group_q.
struct alignas(64) PbJoin {
    int base, x0, nq;               // the list's first token, the first query's place in it
    int own, own_n;
    int common_n, common0, g0, group_q;
    int pad[7];
};

// The plan's parts, in ints from its start
struct PbLayout {
    int64_t rows, items, joins, tasks, toks, total;    // rows: 4 ints each
    int cap_items, cap_joins, cap_tasks, cap_toks;
    int64_t cap_recs;               // records of a kv head
    int slots;                      // blocks per kv head that the device holds at once
};
// header: 0 magic, 1 items, 2 tasks of the join (join * kPbQ + its first query), 3.. the sizes it was made for
constexpr int kPbHeader = 16;

// What a plan can need at most.  Own segments: a row's last may be partly filled;
// common ones: of the rows that share, at least two to a group.  An item is
// ceil(tiles / c) of a segment where c >= all tiles / slots, so all items are at most
// slots + segments, and segments of more than one item have at most 2 slots of them.
static PbLayout pb_layout(int64_t R, int64_t N, int64_t QH, int64_t KVH) {
    PbLayout p{};
    const int64_t G = QH / KVH, NG = N * G, some = NG < kPbAlone * R ? NG : kPbAlone * R, cus = device_cus();
    const int64_t slots = 2 * cus / KVH;
    p.slots = slots < 1 ? 1 : (int)slots;
    p.cap_items = (int)(R + NG / 64 + R / 2 + some / kPbQ + 2) + p.slots;
    const int64_t split = kPbQ < NG ? kPbQ : NG;          // queries of a split segment
    p.cap_joins = (int)(p.slots + R + 1);
    // a query is in one own segment, so in one task at most
    const int64_t tasks = p.slots * split + some + R + 1;
    p.cap_tasks = (int)(tasks < NG ? tasks : NG > 0 ? NG : 1);
    p.cap_toks = (int)some + 1;
    p.cap_recs = 2 * p.slots * split + 2 * some;
    p.rows = kPbHeader;
    p.items = (p.rows + 4 * R + 15) / 16 * 16;
    p.joins = p.items + (int64_t)p.cap_items * (sizeof(PbItem) / 4);
    p.tasks = p.joins + (int64_t)p.cap_joins * (sizeof(PbJoin) / 4);
    p.toks = p.tasks + p.cap_tasks;
    p.total = (p.toks + p.cap_toks + 3) / 4 * 4;
    return p;
}

struct PlanArgs {
    const int32_t* table;
    int64_t table_ld;
    const int32_t* lens;
    const int32_t* fresh;           // new tokens of each row
    int32_t *starts, *rows_of, *positions, *shared;
    int64_t* slots_of;
    int32_t* plan;
    int32_t *limit, *left_out;      // (or NULL)
    PbLayout at;
    int R, N, QH, KVH, G, log_ps, cap, n_pages;
};

// A row's new tokens.  More than the batch holds is one more than it holds (its row
// then does not fit), so that all rows' sum stays within 32 bits.
__device__ __forceinline__ int pb_fresh(const PlanArgs& a, int r) {
    return a.lens[r] < 0 ? 0 : min(max(a.fresh[r], 0), a.N + 1);
}

// ------------------------------------------------------------------ rows

// A wave per row: whether the row has a page for each of its tokens, the ones to come
// included, and with which other row it shares how many leading pages.  Rows that
// start with the same page belong together; the lowest of them leads, found in a hash
// table in LDS that every block fills from all rows' first entries.  A row's state: (the
// leader or -1, whole pages in common with it, pages all there, 0).  Bound by the chain
// first entries, hash, the two rows' entries, 256 of each in flight per wave (64 rows of up to
// 17000 tokens 4.7 us, 256 rows of up to 6600 4.3).
constexpr int kPbHash = 2048;

struct PbHash {
    int key[kPbHash], low[kPbHash];
};

// (at most 1024 different keys in 2048 places: every search ends)
__device__ __forceinline__ int pb_place(int page) { return (int)(((uint32_t)page * 2654435761u) >> 21); }

__device__ __forceinline__ bool pb_candidate(const PlanArgs& a, int m, int n, int page) {
    return m > 0 && (int64_t)m * a.G <= kPbAlone && n >= 1 << a.log_ps && (unsigned)page < (unsigned)a.n_pages;
}

// The table of all rows' first pages (1024 threads)
__device__ __forceinline__ void pb_hash(const PlanArgs& a, PbHash& hash) {
    const int tid = threadIdx.x;
    int page = -1, m = 0, n = -1;
    if (tid < a.R) {
        page = a.table[(int64_t)tid * a.table_ld];
        m = pb_fresh(a, tid);
        n = a.lens[tid];
    }
    for (int i = tid; i < kPbHash; i += 1024) {
        hash.key[i] = -1;
        hash.low[i] = kPbMaxRows;
    }
    __syncthreads();
    if (pb_candidate(a, m, n, page)) {
        for (int h = pb_place(page);; h = (h + 1) & (kPbHash - 1)) {
            const int was = atomicCAS(&hash.key[h], -1, page);
            if (was == -1 || was == page) {
                atomicMin(&hash.low[h], tid);
                break;
            }
        }
    }
    __syncthreads();
}

// Row r's state, by a wave
__device__ __forceinline__ int4 pb_row(const PlanArgs& a, const PbHash& hash, int r) {
    const int lane = threadIdx.x & 63, PS = 1 << a.log_ps, n = a.lens[r], m = pb_fresh(a, r);
    const int32_t* row = a.table + (int64_t)r * a.table_ld;
    const int first = row[0];
    int lead = -1;
    if (pb_candidate(a, m, n, first)) {
        int h = pb_place(first);
        while (hash.key[h] != first) h = (h + 1) & (kPbHash - 1);
        lead = hash.low[h];
    }
    lead = __builtin_amdgcn_readfirstlane(lead);
    const bool fits = n >= 0 && n <= a.cap && m <= a.cap - n;
    const int need = m > 0 && fits ? (n + m + PS - 1) >> a.log_ps : 0, whole = lead >= 0 ? n >> a.log_ps : 0;
    const int32_t* other = a.table + (int64_t)max(lead, 0) * a.table_ld;
    bool there = fits;
    int same = whole;
    for (int c0 = 0; c0 < need; c0 += 256) {
        int v[4], w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int c = min(c0 + 64 * u + lane, need - 1);         // (a condition would wait for each load)
            v[u] = row[c];
            w[u] = other[c];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            there &= !__any((unsigned)v[u] >= (unsigned)a.n_pages);
            const unsigned long long differ = __ballot(c0 + 64 * u + lane < whole && v[u] != w[u]);
            if (differ) same = min(same, c0 + 64 * u + (int)__ffsll(differ) - 1);
        }
    }
    return make_int4(lead, same, there, 0);
}

__global__ void __launch_bounds__(1024)
paged_rows_kernel(PlanArgs a) {
    __shared__ PbHash hash;
    pb_hash(a, hash);
    const int r = blockIdx.x * 16 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (r >= a.R) return;
    const int4 s = pb_row(a, hash, r);
    if ((threadIdx.x & 63) == 0) *reinterpret_cast<int4*>(a.plan + a.at.rows + 4 * r) = s;
}

// ------------------------------------------------------------------ plan

// Exclusive scan of N counts over the NT threads of a block; total: their sums.
template <int NT, int N>
__device__ __forceinline__ void pb_scan(const int (&v)[N], int* waves, int (&before)[N], int (&total)[N]) {
    constexpr int NW = NT / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int incl[N];
    __syncthreads();                                 // the previous use of `waves` is over
#pragma unroll
    for (int k = 0; k < N; ++k) {
        incl[k] = wave_scan_int(v[k]);
        if constexpr (NW == 1) {
            total[k] = __builtin_amdgcn_readlane(incl[k], 63);
            before[k] = incl[k] - v[k];
        } else if (lane == 63) {
            waves[wave * N + k] = incl[k];
        }
    }
    if constexpr (NW > 1) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int mine = lane < NW ? waves[lane * N + k] : 0;
            const int upto = wave_scan_int(mine);
            total[k] = __builtin_amdgcn_readlane(upto, NW - 1);
            before[k] = __builtin_amdgcn_readlane(upto - mine, __builtin_amdgcn_readfirstlane(wave)) + incl[k] - v[k];
        }
    }
}

// The last of `n` ascending values that is at most x (values[0] <= x)
__device__ __forceinline__ int pb_find(const int* values, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (values[mid] <= x) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// The rows' states as paged_rows_kernel finds them, by a block of NT threads at once: a
// thread per row for the leaders, per table entry for the pages.
template <int NT>
__device__ __forceinline__ int4 pb_states(const PlanArgs& a, int m) {
    __shared__ __align__(16) int page_of[NT], need_of[NT], whole_of[NT], same_of[NT], lacks[NT];
    const int r = threadIdx.x, PS = 1 << a.log_ps;
    int n = -1, page = -1 - r;                       // (no two rows that are no candidates have the same)
    if (r < a.R) {
        n = a.lens[r];
        const int first = a.table[(int64_t)r * a.table_ld];
        if (pb_candidate(a, m, n, first)) page = first;
    }
    const bool fits = n >= 0 && n <= a.cap && m <= a.cap - n;
    page_of[r] = page;
    need_of[r] = m > 0 && fits ? (n + m + PS - 1) >> a.log_ps : 0;
    whole_of[r] = same_of[r] = page >= 0 ? n >> a.log_ps : 0;
    lacks[r] = 0;
    __syncthreads();
    int lead = page >= 0 ? r : -1;
    if (page >= 0) {
#pragma unroll 4
        for (int i = 0; i < r; i += 4) {
            const int4 q = *reinterpret_cast<const int4*>(page_of + i);
            if (q.w == page && i + 3 < lead) lead = i + 3;
            if (q.z == page && i + 2 < lead) lead = i + 2;
            if (q.y == page && i + 1 < lead) lead = i + 1;
            if (q.x == page && i < lead) lead = i;
        }
    }
    __syncthreads();
    page_of[r] = lead;
    __syncthreads();
    const int MP = a.cap >> a.log_ps, entries = a.R * MP;
    const float per = 1.0f / (float)MP;              // (entries are few: the quotient is off by one at most)
    for (int i0 = r; i0 < entries; i0 += 4 * NT) {
        // (all of a round's entries are loaded, needed or not: a condition would wait for each)
        int v[4], w[4], row[4], col[4], lead_row[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = min(i0 + u * NT, entries - 1);
            row[u] = (int)((float)i * per);
            col[u] = i - row[u] * MP;
            if (col[u] < 0) --row[u], col[u] += MP;
            if (col[u] >= MP) ++row[u], col[u] -= MP;
            lead_row[u] = max(page_of[row[u]], 0);
            v[u] = a.table[(int64_t)row[u] * a.table_ld + col[u]];
            w[u] = a.table[(int64_t)lead_row[u] * a.table_ld + col[u]];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (col[u] < need_of[row[u]] && (unsigned)v[u] >= (unsigned)a.n_pages) lacks[row[u]] = 1;
            if (col[u] < whole_of[row[u]] && v[u] != w[u]) atomicMin(&same_of[row[u]], col[u]);
        }
    }
    __syncthreads();
    return make_int4(lead, same_of[r], fits && lacks[r] == 0, 0);
}

// Block 0: groups, segments, items, joins.  The others, NT flat tokens each: the
// tokens' rows, positions and slots.  Both begin with a scan over the rows' counts.
// Block 0 is one block because each stage needs the whole of the one before; it is
// bound by their latency, a pass over the rows or the segments with a block scan each.
// ALONE: of few table entries every block finds the states itself, and the launch before is
// saved.  NT: at least as many threads as rows; a barrier of fewer waves is a shorter one
// (4 rows by one wave 6.2 us, by 16 with the launch before 9.2; 32 rows by four waves 11.1, 64
// and 256 rows by 16 waves 9 to 11 behind the launch before).
template <int NT, bool ALONE>
__global__ void __launch_bounds__(NT)
paged_plan_kernel(PlanArgs a) {
    __shared__ __align__(16) int first[NT], m_of[NT], lead_of[NT];
    __shared__ int gpages[NT], gtoks[NT], gbase[NT], pbase[NT], sbase[NT];
    __shared__ int rowx[NT], grec[NT], gend[NT];
    __shared__ int waves[NT / 64 * 4];
    const int tid = threadIdx.x, r = tid, PS = 1 << a.log_ps;
    int m = 0;
    int4 info = make_int4(-1, 0, 0, 0);
    if (r < a.R) m = pb_fresh(a, r);
    if constexpr (ALONE) info = pb_states<NT>(a, m);
    else if (r < a.R) info = *reinterpret_cast<const int4*>(a.plan + a.at.rows + 4 * r);
    int m1[1] = {m}, start1[1], all1[1];
    pb_scan<NT, 1>(m1, waves, start1, all1);
    const int start = start1[0];
    const bool ok = m > 0 && info.z != 0 && start + m <= a.N;
    first[r] = r < a.R ? start : 0x7fffffff;
    m_of[r] = ok ? m : 0;
    if (blockIdx.x > 0) {
        __syncthreads();
        const int t = (blockIdx.x - 1) * NT + tid;
        if (t >= a.N) return;
        int row = -1, pos = -1;
        int64_t slot = -1;
        if (t < all1[0]) {
            row = pb_find(first, a.R, t);
            pos = a.lens[row] + t - first[row];
            if (m_of[row] > 0)
                slot = ((int64_t)a.table[(int64_t)row * a.table_ld + (pos >> a.log_ps)] << a.log_ps) + (pos & (PS - 1));
            if (pos < 0) pos = 0x7fffffff;           // (a row that has no room for its tokens)
        }
        a.rows_of[t] = row;
        a.positions[t] = pos;
        a.slots_of[t] = slot;
        return;
    }
    if (r < a.R) a.starts[r] = start;
    if (r == 0) a.starts[a.R] = all1[0];
    if (m > 0 && a.limit != nullptr) a.limit[r] = ok ? 0x7fffffff : 0;
    if (m > 0 && !ok && a.left_out != nullptr) atomicAdd(a.left_out, 1);

    // groups: rows of one leader; what all of them have in common
    const int lead = ok && info.x >= 0 ? info.x : -1;
    lead_of[r] = lead;
    gpages[r] = 0x7fffffff;
    gtoks[r] = 0;
    gend[r] = 0;
    gbase[r] = 0;                                    // rows of the group, for now
    __syncthreads();
    if (lead >= 0) {
        atomicMin(&gpages[lead], info.y);
        atomicAdd(&gtoks[lead], m);
        atomicAdd(&gbase[lead], 1);
        atomicMax(&gend[lead], start + m);
    }
    __syncthreads();
    // common positions of the group that row r leads
    const bool pays = gbase[r] >= 2 && gpages[r] << a.log_ps >= kPbShare;
    const int npre = pays ? (gtoks[r] * a.G + kPbQ - 1) / kPbQ : 0;
    const int64_t queries = ok ? (int64_t)m * a.G : 0;
    __syncthreads();
    if (!pays) gpages[r] = 0;
    int four[4] = {pays ? gtoks[r] : 0, npre, (int)((queries + kPbQ - 1) / kPbQ), (int)((queries + 63) / 64)}, before[4], total[4];
    pb_scan<NT, 4>(four, waves, before, total);
    // own segments of 64 queries where those fill the device whole and ones of 128 would have to be split
    const bool small = total[2] < a.at.slots && total[3] >= a.at.slots;
    const int own_q = small ? 64 : kPbQ, n_own = small ? total[3] : total[2];
    gbase[r] = before[0];
    pbase[r] = before[1];
    sbase[r] = total[1] + (small ? before[3] : before[2]);
    __syncthreads();
    const int shared = lead >= 0 ? gpages[lead] << a.log_ps : 0;
    int ahead = 0;                                   // tokens of the group's rows before this one
    if (shared > 0) {
#pragma unroll 4
        for (int i = lead & ~3; i < r; i += 4) {     // (rows in front of the leader have others)
            const int4 l = *reinterpret_cast<const int4*>(lead_of + i), n = *reinterpret_cast<const int4*>(m_of + i);
            ahead += (l.x == lead ? n.x : 0) + (l.y == lead && i + 1 < r ? n.y : 0) + (l.z == lead && i + 2 < r ? n.z : 0) +
                     (l.w == lead && i + 3 < r ? n.w : 0);
        }
        for (int i = 0; i < m; ++i) a.plan[a.at.toks + gbase[lead] + ahead + i] = start + i;
    }
    rowx[r] = ahead;
    if (r < a.R) a.shared[r] = shared;
    __syncthreads();

    const int nseg = total[1] + n_own;
    // a segment as one item; *of: its row or its group's leader, *tiles_of: its tiles
    auto segment = [&](int i, int* of, int* tiles_of) __attribute__((always_inline)) {
        PbItem s{};
        const bool common = i < total[1];
        const int row = pb_find(common ? pbase : sbase, a.R, i);
        const int x0 = common ? (i - pbase[row]) * kPbQ : (i - sbase[row]) * own_q;
        *of = row;
        s.row = row;
        s.x0 = x0;
        if (common) {
            s.nq = min(kPbQ, gtoks[row] * a.G - x0);
            s.kind = gend[row] - first[row] == gtoks[row] ? kPbRun : kPbList;
            s.base = s.kind == kPbRun ? first[row] : gbase[row];
            s.key0 = 0;
            s.key1 = gpages[row] << a.log_ps;
            s.lens = s.key1;
        } else {
            s.kind = kPbOwn;
            s.nq = (int)min((int64_t)own_q, (int64_t)m_of[row] * a.G - x0);
            s.base = first[row];
            s.lens = a.lens[row];
            const int l = lead_of[row];
            s.key0 = l >= 0 ? gpages[l] << a.log_ps : 0;
            s.key1 = s.lens + (x0 + s.nq - 1) / a.G + 1;
        }
        *tiles_of = (s.key1 - s.key0 + kPbTile - 1) / kPbTile;
        return s;
    };
    auto chunks = [&](int n, int chunk) { return (n + chunk - 1) / chunk; };
    // (up to 2^24 segments of 2^18 tiles: the sum's upper and lower 20 bits apart)
    int64_t mine = 0, sixteens = 0;                  // tiles; tiles times blocks of 16 queries
    int of = 0, s_tiles = 0;
    PbItem s{};                                      // the thread's first segment, often its only one
    for (int i = tid; i < nseg; i += NT) {
        int n;
        const PbItem g = segment(i, &of, &n);
        if (i == tid) {
            s = g;
            s_tiles = n;
        }
        mine += n;
        sixteens += (int64_t)n * ((g.nq + 15) / 16);
    }
    const int of0 = nseg <= NT ? of : 0;
    // the common segments' records come first: a group's begin behind those of the groups before it
    int sum[4] = {(int)(mine >> 20), (int)(mine & 0xfffff), (int)(sixteens >> 20), (int)(sixteens & 0xfffff)}, none[4], tiles[4];
    pb_scan<NT, 4>(sum, waves, none, tiles);
    const int64_t all_tiles = ((int64_t)tiles[0] << 20) + tiles[1];
    // An item has at least the tiles that fill the device.  It leaves a record per query, which
    // is written and read at the copy's rate by all blocks together, while a tile is
    // one block's time: c tiles and work / c records take least where c^2 is their ratio.
    // That is a rule of thumb: it does not know how many whole times the items fill the device, and
    // `fill` counts a tile of few queries like one of 128, so times jump with c rather than
    // follow a curve.  (kPbRecord 1.5e-4 / 2.5e-4 / 4e-4 / 1e-3, items and join, us: 64 rows behind
    // 16384 71.1 / 70.5 / 62.5 / 76.2, with c 11 / 11 / 14 / 23, the first two what fills the device;
    // 4 x 12 behind 1500 30.4 / 32.5 / 33.8 / 38.4, c 4 / 6 / 7 / 12; 2 x 16 behind 2048 21.0 / 20.5 /
    // 19.1 / 19.4.  4e-4 is the best of them for two of the three and costs the third a tenth.)
    const float ratio = kPbRecord * (float)a.KVH * 16.0f * ((float)tiles[2] * 1048576.0f + (float)tiles[3]);
    const int64_t fill = (all_tiles + a.at.slots - 1) / a.at.slots;
    const int chunk = max(max(kPbLeast, (int)sqrtf(ratio)), (int)min(fill, (int64_t)1 << 30));
    if (total[1] > 0) {
        const int positions = gpages[r] << a.log_ps;
        int recs[1] = {pays ? gtoks[r] * a.G * chunks((positions + kPbTile - 1) / kPbTile, chunk) : 0}, at1[1], all_r[1];
        pb_scan<NT, 1>(recs, waves, at1, all_r);
        grec[r] = at1[0];
        __syncthreads();
    }
    int item0 = 0, rec0 = 0, join0 = 0, task0 = 0;
    for (int i0 = 0; i0 < nseg; i0 += NT) {
        const int i = i0 + tid;
        const bool in = i < nseg;
        of = of0;
        if (nseg > NT && in) s = segment(i, &of, &s_tiles);
        int want[4] = {0, 0, 0, 0}, at[4], sums[4];
        const int n = chunks(s_tiles, chunk);
        const bool shares = s.kind == kPbOwn && s.key0 > 0, rec = n > 1 || s.kind != kPbOwn || shares;
        const int common_n = shares ? chunks((s.key0 + kPbTile - 1) / kPbTile, chunk) : 0;
        if (in) {
            want[0] = rec ? n * s.nq : 0;
            want[1] = rec && s.kind == kPbOwn;
            want[2] = n;
            want[3] = !want[1] ? 0 : n + common_n <= kPbFew ? (s.nq + 3) / 4 : s.nq;
        }
        pb_scan<NT, 4>(want, waves, at, sums);
        if (in) {
            const int own = rec0 + at[0];
            if (want[1]) {
                PbJoin t{};
                t.base = s.base;
                t.x0 = s.x0;
                t.nq = s.nq;
                t.own = own;
                t.own_n = n;
                if (shares) {
                    const int l = lead_of[of];
                    t.common_n = common_n;
                    t.common0 = grec[l];
                    t.g0 = rowx[of] * a.G + s.x0;
                    t.group_q = gtoks[l] * a.G;
                }
                reinterpret_cast<PbJoin*>(a.plan + a.at.joins)[join0 + at[1]] = t;
            }
        }
        // the items of a segment and the tasks of a join: by its thread, and by the wave where few
        // of its threads have many (1 row of 16384: 10.1 -> 6.7 us)
        auto put = [&](PbItem g, int k, int n, int own, int at_item) __attribute__((always_inline)) {
            const int q = g.tile1 / n, more = g.tile1 - q * n;       // (tile1: all its tiles)
            g.tile0 = k * q + min(k, more);
            g.tile1 = (k + 1) * q + min(k + 1, more);
            if (own >= 0) g.rec = own + k * g.nq;
            reinterpret_cast<PbItem*>(a.plan + a.at.items)[at_item + k] = g;
        };
        s.tile1 = s_tiles;
        s.rec = -1;
        const int own = rec ? rec0 + at[0] : -1, item = item0 + at[2], task = task0 + at[3];
        const int code = (join0 + at[1]) * kPbQ, step = n + common_n <= kPbFew ? 4 : 1, tasks = want[3];
        constexpr int kMany = 8, kFewOf = 4;
        const int lane = tid & 63;
        unsigned long long big = __ballot(in && n > kMany);
        if (__popcll(big) > kFewOf) big = 0;
        if (in && !(big >> lane & 1))
            for (int k = 0; k < n; ++k) put(s, k, n, own, item);
        while (big) {
            const int src = __builtin_amdgcn_readfirstlane(__ffsll(big) - 1);
            big &= big - 1;
            PbItem g = s;
            int* p = reinterpret_cast<int*>(&g);
#pragma unroll
            for (int i = 0; i < 11; ++i) p[i] = __builtin_amdgcn_readlane(p[i], src);
            const int gn = __builtin_amdgcn_readlane(n, src), go = __builtin_amdgcn_readlane(own, src), gi = __builtin_amdgcn_readlane(item, src);
            for (int k = lane; k < gn; k += 64) put(g, k, gn, go, gi);
        }
        big = __ballot(tasks > kMany);
        if (__popcll(big) > kFewOf) big = 0;
        if (!(big >> lane & 1))
            for (int k = 0; k < tasks; ++k) a.plan[a.at.tasks + task + k] = code + step * k;
        while (big) {
            const int src = __builtin_amdgcn_readfirstlane(__ffsll(big) - 1);
            big &= big - 1;
            const int gn = __builtin_amdgcn_readlane(tasks, src), gt = __builtin_amdgcn_readlane(task, src);
            const int gc = __builtin_amdgcn_readlane(code, src), gs = __builtin_amdgcn_readlane(step, src);
            for (int k = lane; k < gn; k += 64) a.plan[a.at.tasks + gt + k] = gc + gs * k;
        }
        rec0 += sums[0];
        join0 += sums[1];
        item0 += sums[2];
        task0 += sums[3];
    }
    if (tid == 0) {
        a.plan[0] = kPbMagic;
        a.plan[1] = item0;
        a.plan[2] = task0;
        a.plan[3] = a.R;
        a.plan[4] = a.N;
        a.plan[5] = a.QH;
        a.plan[6] = a.KVH;
        a.plan[7] = a.cap;
        a.plan[8] = a.log_ps;
        a.plan[9] = a.at.slots;
        a.plan[10] = a.n_pages;
    }
}

// ------------------------------------------------------------------ a layer's step

template <typename T>
struct BatchArgs {
    const T* qkv;                   // projection rows [q | k | v] of the flat tokens
    int64_t qkv_ld;
    T* kp;
    T* vp;
    int64_t ps_page, ps_tok, ps_head;
    const int32_t* table;
    int64_t table_ld;
    const int32_t *positions, *rows_of;
    const int64_t* slots_of;
    const float *cosv, *sinv;
    T *q_out, *c_out, *k_out;
    int64_t out_ld;
    const int32_t* plan;
    PbLayout at;
    uint8_t* odd;                   // tokens whose k or v holds an infinity or NaN
    float* rec;                     // [KVH, cap_recs, 2 HD], then [KVH, cap_recs, 2]
    int64_t rec_ml;
    int R, N, QH, KVH, G, HD, log_ps, cap, n_pages, n_pos;
    float qscale;
};

// Whether the plan is one of these sizes (another one's numbers could lie anywhere)
template <typename T>
__device__ __forceinline__ bool plan_fits(const BatchArgs<T>& a) {
    const int32_t* h = a.plan;
    return h[0] == kPbMagic && h[3] == a.R && h[4] == a.N && h[5] == a.QH && h[6] == a.KVH && h[7] == a.cap &&
           h[8] == a.log_ps && h[9] == a.at.slots && h[10] == a.n_pages;
}

template <typename T, int E>
__device__ __forceinline__ void load_e(const T* p, float (&v)[E]) {
    if constexpr (E == 8) {
        Vec8<T>::load(p, v);
    } else if constexpr (sizeof(T) == 4) {
        const float4 w = *reinterpret_cast<const float4*>(p);
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    } else {
        RowIO<T, 4>::load(p, v);
    }
}
template <typename T, int E>
__device__ __forceinline__ void store_e(T* p, const float (&v)[E]) {
    if constexpr (E == 8) {
        Vec8<T>::store(p, v);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        T t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) st(t + e, v[e]);
        *reinterpret_cast<uint2*>(p) = make_uint2((uint32_t)t[0].x | ((uint32_t)t[1].x << 16),
                                                  (uint32_t)t[2].x | ((uint32_t)t[3].x << 16));
    }
}

// A block per token: q and k roped and rounded, q to q_out, k and v into the token's
// slot.  A thread takes E elements of a head and their partners half a head on, so that
// each is loaded once.  Tokens behind the last give zeros, tokens of a row without room
// or a page NaN; both are done here.  A copy with a little arithmetic.  Of wide tokens bound by the
// bytes in and out (5139 tokens of 48 heads of 128 25.4 us, 5.0 TB/s), of few tokens by one
// load after the other (32 tokens 4.8).  Many narrow tokens are bound by neither: of 12 heads of 96 84
// threads of a block have work, a piece each, and what counts is the blocks' number times
// their latency (4096 tokens 11.1 us in bf16, 1.7 TB/s, and 11.7 in fp32).
template <typename T, int E>
__global__ void __launch_bounds__(256)
paged_append_kernel(BatchArgs<T> a) {
    const int t = blockIdx.x, tid = threadIdx.x;
    const int row = a.rows_of[t], pos = a.positions[t], half = a.HD / 2;
    const int64_t slot = a.slots_of[t], page = slot >> a.log_ps;
    const bool fits = plan_fits(a);
    const bool in = fits && row >= 0 && slot >= 0 && page < a.n_pages, turned = in && pos < a.n_pos && pos >= 0;
    if (!turned) {
        const float fill = row >= 0 || !fits ? NAN : 0.0f;
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = fill;
        for (int i = tid; i < a.QH * a.HD / E; i += 256) {
            const int h = i * E / a.HD, d = i * E - h * a.HD;
            store_e<T, E>(a.q_out + ((int64_t)t * a.QH + h) * a.HD + d, v);
            // (the items write those of tokens that the plan has)
            if (in) continue;
            store_e<T, E>(a.c_out + t * a.out_ld + i * E, v);
            if (a.k_out != nullptr) store_e<T, E>(a.k_out + t * a.out_ld + i * E, v);
        }
        if (tid == 0) a.odd[t] = 1;
        return;
    }
    const T* x = a.qkv + t * a.qkv_ld;
    const float *cr = a.cosv + (int64_t)pos * a.HD, *sr = a.sinv + (int64_t)pos * a.HD;
    const int64_t at = page * a.ps_page + (slot & ((1 << a.log_ps) - 1)) * a.ps_tok;
    const int per = half / E, turns = (a.QH + a.KVH) * per, vper = a.HD / E;
    bool odd = false;
    for (int i = tid; i < turns + a.KVH * vper; i += 256) {
        if (i < turns) {
            const int h = i / per, d = (i - h * per) * E;
            float u[E], w[E], c0[E], s0[E], c1[E], s1[E], lo[E], hi[E];
            load_e<T, E>(x + h * a.HD + d, u);
            load_e<T, E>(x + h * a.HD + d + half, w);
            load_e<float, E>(cr + d, c0);
            load_e<float, E>(sr + d, s0);
            load_e<float, E>(cr + d + half, c1);
            load_e<float, E>(sr + d + half, s1);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                lo[e] = turn<T>(u[e], c0[e], -w[e], s0[e]);
                hi[e] = turn<T>(w[e], c1[e], u[e], s1[e]);
            }
            T* out = h < a.QH ? a.q_out + ((int64_t)t * a.QH + h) * a.HD : a.kp + at + (h - a.QH) * a.ps_head;
            store_e<T, E>(out + d, lo);
            store_e<T, E>(out + d + half, hi);
            if (h >= a.QH) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    odd |= !(fabsf(round_to<T>(lo[e])) < INFINITY) || !(fabsf(round_to<T>(hi[e])) < INFINITY);
            }
        } else {
            const int h = (i - turns) / vper, d = (i - turns - h * vper) * E;
            float u[E];
            load_e<T, E>(x + (a.QH + a.KVH + h) * a.HD + d, u);
            store_e<T, E>(a.vp + at + h * a.ps_head + d, u);
#pragma unroll
            for (int e = 0; e < E; ++e) odd |= !(fabsf(u[e]) < INFINITY);
        }
    }
    odd = __syncthreads_or(odd);
    if (tid == 0) a.odd[t] = odd;
}

// What a block works on: an item of a kv head, or nothing.  Item blockIdx.x / KVH of kv head
// blockIdx.x % KVH: blocks go to the XCDs in turn, so that 8 kv heads have an XCD's L2 each
// for their keys, and fewer share them among several.
struct PbWork {
    PbItem s;
    int kvh;
    bool any;
};

template <typename T>
__device__ __forceinline__ PbWork pb_work(const BatchArgs<T>& a) {
    PbWork w;
    const int item = blockIdx.x / a.KVH;
    // (the item is loaded with the count that says whether it is one)
    w.s = reinterpret_cast<const PbItem*>(a.plan + a.at.items)[item];
    w.any = item < a.plan[1] && plan_fits(a);
    w.kvh = blockIdx.x - item * a.KVH;
    int* p = reinterpret_cast<int*>(&w.s);           // the same in all lanes, which the compiler may not see
#pragma unroll
    for (int i = 0; i < 11; ++i) p[i] = __builtin_amdgcn_readfirstlane(p[i]);
    return w;
}

// Flat token of query x of a segment
template <typename T>
__device__ __forceinline__ int pb_token(const BatchArgs<T>& a, const PbItem& s, int x) {
    const int i = s.base + (s.x0 + x) / a.G;
    return s.kind == kPbList ? a.plan[a.at.toks + i] : i;
}

// Positions that query x sees: all of a common segment, up to itself of its own row's
template <typename T>
__device__ __forceinline__ int pb_sees(const BatchArgs<T>& a, const PbItem& s, int x) {
    return s.kind != kPbOwn ? s.key1 : s.lens + (s.x0 + x) / a.G + 1;
}

// Infinities and NaN.  A weight of zero does not silence them in a matrix product, so a
// new token that holds one must not enter the products of queries that do not see it.
// Where a block has such a token (pb_odd), the products leave out what is not finite in
// rows that not every query sees, and the item's end adds it to the sums of the
// queries that do (pb_poison): an infinity of v is the sum's, one of k (whose score is NaN
// or an infinity, and 0 times an infinity) is NaN.  Such tokens lie behind the first query's
// (pb_new), and only the item that holds a token's position adds it: in another one a query
// that sees it may see nothing at all, and the join would take the infinity times zero.
// What every query of the block sees, tokens of earlier steps among it, stays in the products: an
// infinity of v there is the sum's where its weight is not zero in the type that the product
// takes, and NaN where it is.
struct PbNew {
    int first, last;                // new tokens of the row, from 0
};

// New tokens whose positions the item holds and that some of the block's queries do not see
template <typename T>
__device__ __forceinline__ PbNew pb_new(const BatchArgs<T>& a, const PbItem& s) {
    const int k0 = s.key0 + s.tile0 * kPbTile, kend = min(s.key1, s.key0 + s.tile1 * kPbTile);
    return {max(s.x0 / a.G + 1, k0 - s.lens), min((s.x0 + s.nq - 1) / a.G, kend - 1 - s.lens)};
}

template <typename T>
__device__ __forceinline__ bool pb_odd(const BatchArgs<T>& a, const PbItem& s) {
    bool odd = false;
    if (s.kind == kPbOwn) {
        const PbNew n = pb_new(a, s);
        for (int i = n.first + threadIdx.x; i <= n.last; i += 256) odd |= a.odd[s.base + i] != 0;
    }
    return odd;
}

template <typename T>
__device__ __noinline__ float pb_poison(const T* pool, const uint8_t* odd, const int32_t* row, int64_t ps_page, int64_t ps_tok,
                                        int lens, int log_ps, int n_pages, int first, int last, bool nan) {
    float c = 0.0f;
    for (int i = first; i <= last; ++i) {
        if (odd[i] == 0) continue;
        const int t = lens + i, page = row[t >> log_ps];
        if ((unsigned)page >= (unsigned)n_pages) continue;
        const float v = ld(pool + (int64_t)page * ps_page + (int64_t)(t & ((1 << log_ps) - 1)) * ps_tok);
        if (!(fabsf(v) < INFINITY)) c += nan ? NAN : v;
    }
    return c;
}

// 16-bit elements that are not finite as zeros
template <typename T>
__device__ __forceinline__ gqa_u4 pb_finite(gqa_u4 w) {
    constexpr uint32_t E = std::is_same<T, bf16_t>::value ? 0x7f80u : 0x7c00u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((w[i] & E) == E) w[i] &= 0xffff0000u;
        if ((w[i] & (E << 16)) == E << 16) w[i] &= 0xffffu;
    }
    return w;
}

// The end of an item, for 16 queries of each of its four waves: their (m, l, C, Kctx) joined
// into records, or into the outputs where the queries have no other part.  part(w): the sums of
// wave w's queries as its lanes hold them, C then Kctx, four queries' of one dimension
// side by side.  QW waves stand side by side: wave w's queries begin at first +
// (w % QW) apart, and waves w, w + QW, .. have the same.  First a thread per query finds the
// factors of its parts and where it goes, then every thread takes four queries' sums of one
// dimension (4 tokens behind 333 8.3 -> 7.2 us for the kernel, 8 x 4 behind 2048 12.0 -> 11.0,
// 2 x 16 behind 2048 16.7 -> 15.1, against factors and destinations found by every thread
// in a loop that held the rare cases).
struct PbEnd {
    float2 ml[4][16];
    __align__(16) float factor[4][64];
    int64_t to[64];                                  // element of the outputs (< 0: none) or record
    int last[64];                                    // the query's token in the row's new ones
};

template <int HDP, bool KCTX, int QW, typename T, typename P>
__device__ __forceinline__ void pb_finish(const BatchArgs<T>& a, const PbWork& w, int first, int apart, bool odd, PbEnd& end, P part) {
    const PbItem& s = w.s;
    constexpr int KW = 4 / QW, D = KCTX ? 2 * HDP : HDP;
    const int tid = threadIdx.x;
    __syncthreads();                                 // the parts are written
    if (tid < 16 * QW) {
        const int x = first + (tid >> 4) * apart + (tid & 15);
        float m = -INFINITY, l = 0.0f, f[KW];
#pragma unroll
        for (int g = 0; g < KW; ++g) m = fmaxf(m, end.ml[(tid >> 4) + QW * g][tid & 15].x);
#pragma unroll
        for (int g = 0; g < KW; ++g) {
            const float2 p = end.ml[(tid >> 4) + QW * g][tid & 15];
            f[g] = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(p.x - m);
            l = fmaf(p.y, f[g], l);
        }
        const float inv = s.rec < 0 ? 1.0f / l : 1.0f;
#pragma unroll
        for (int g = 0; g < KW; ++g) end.factor[g][tid] = f[g] * inv;
        int64_t to = -1;
        if (x < s.nq) {
            const int i = (s.x0 + x) / a.G, h = w.kvh * a.G + s.x0 + x - i * a.G;
            if (s.rec < 0) {
                to = (int64_t)pb_token(a, s, x) * a.out_ld + (int64_t)h * a.HD;
            } else {
                to = w.kvh * a.at.cap_recs + s.rec + x;
                *reinterpret_cast<float2*>(a.rec + a.rec_ml + 2 * to) = make_float2(m, l);
            }
            end.last[tid] = i;
        }
        end.to[tid] = to;
    }
    __syncthreads();
    // the usual loop has neither the rare tokens nor the other destination in it: a block runs
    // through this code once, and what it costs is fetching it
    auto sums = [&](auto poison, auto out) {
        const PbNew mine = pb_new(a, s);
#pragma unroll 1
        for (int k = tid; k < 4 * QW * D; k += 256) {
            const int four = k / D, dd = k - four * D, which = dd >= HDP, d = dd - which * HDP, w0 = four >> 2;
            pg_f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int g = 0; g < KW; ++g) {
                // queries 4 (four % 4) .. + 3, dimension d: lane 16 (four % 4) + d % 16
                const pg_f32x4 v = reinterpret_cast<const pg_f32x4*>(part(w0 + QW * g))[(which * (HDP / 16) + (d >> 4)) * 64 + (four & 3) * 16 + (d & 15)];
                c += v * *reinterpret_cast<const pg_f32x4*>(&end.factor[g][4 * four]);
            }
            if (HDP > a.HD && d >= a.HD && out) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t to = end.to[4 * four + i];
                if (to < 0) continue;
                if (poison && d < a.HD)
                    c[i] += pb_poison((which ? a.kp : a.vp) + w.kvh * a.ps_head + d, a.odd + s.base, a.table + (int64_t)s.row * a.table_ld,
                                      a.ps_page, a.ps_tok, s.lens, a.log_ps, a.n_pages, mine.first, min(mine.last, end.last[4 * four + i]), which);
                if (out) st((which ? a.k_out : a.c_out) + to + d, c[i]);
                else a.rec[to * 2 * HDP + dd] = c[i];
            }
        }
    };
    using Yes = std::true_type;
    using No = std::false_type;
    if (odd) s.rec < 0 ? sums(Yes{}, Yes{}) : sums(Yes{}, No{});
    else s.rec < 0 ? sums(No{}, Yes{}) : sums(No{}, No{});
}

// ------------------------------------------------------------------ matrix-core form
// 16-bit types, HD 32 / 64 / 96 / 128.  Four waves stream 64 positions per step through
// NS LDS stages that loads fill directly, one barrier per step; a 16-position quarter of
// a tile lies in one page (pages hold a multiple of 16 positions), staged by one wave, so
// its base and its bound are scalar: rows past the item's end land as zeros.  QW waves
// side by side take NQ times 16 queries each, and the KW = 4 / QW groups of them a quarter,
// half or all of the positions, so that a decode step's few queries use all waves too:
//   queries      QW NQ KW
//   1 .. 16       1  1  4
//   17 .. 32      2  1  2
//   33 .. 64      2  2  2
//   65 .. 128     4  2  1
// Two query blocks per wave share every K and V fragment's LDS read.  S^T = K Q^T, P from
// the score registers, C = P V and Kctx = P K through the transposing LDS read.  A lane's
// sum of weights is its own until the end, and the reference of the exponents is looked at
// lane by lane: the lanes of a column meet only where it has to rise.
//
// Of long shared runs and of prompts bound by the matrix products and what feeds them: 5139
// tokens of 32 heads of 128 in 284 us, 740 TFLOP/s (the 8192^3 product 1135), in half 323; without Kctx
// 212; 62 rows behind 16384 51.8 us, 486 TFLOP/s, of which the records' 40 MB written at once are some 8
// (without Kctx 41.5); 32 x 128 tokens behind 1920 of 8 heads of 96 58.2 us, 645 TFLOP/s.  Of few rows by the
// chain item, page, first tile, sums: 7.2 us (4 rows behind 333), 11.1 (8 x 4 behind 2048, 1.4 TB/s).
template <int HD> constexpr int pb_stages() { return HD <= 96 ? 3 : 2; }

// Where a row's 16-byte pieces lie in a stage: piece c of row r at c ^ swz(r), so that both
// fragment reads spread over the banks.  Rows of 4 or 12 pieces go by attn_tile.h's two bits;
// of 8 and 16, where rows begin on the same banks, by three and four.  LDS cycles of a 16-byte
// read and of a transposing one, timed over such maps with 16 waves: 3.7 and 2.05 at best
// (the two bits in rows of 16 pieces: 10.9 and 4.9; no swizzle: 19.3 and 9.0).
template <int CPR>
struct PbLane {
    static constexpr bool kXor = CPR == 8 || CPR == 16;
    // nibble r: bits (r2, r1, r1^r2, r0^r3) of rows of 16 pieces, (r0^r1, r1, r1^r2) of 8
    static constexpr uint64_t kMap = CPR == 16 ? 0x3b5d6e08b3d5e680ull : 0x2354671023546710ull;
    const TileLane<CPR> lane;
    uint32_t s_at, t_at;
    __device__ __forceinline__ static int swz(int r) {
        if constexpr (kXor) return (int)(kMap >> (4 * (r & 15))) & 15;
        else return kv_swz(r);
    }
    __device__ __forceinline__ PbLane(int lq, int lr) : lane(lq, lr) {
        const int row = 4 * lq + (lr >> 2);
        s_at = (uint32_t)(lr * CPR + (lq ^ swz(lr))) * 16;
        t_at = (uint32_t)(row * CPR + (((lr & 3) >> 1) ^ swz(row))) * 16 + 8 * (lr & 1);
    }
    // the A operand of S^T: row 16 hf + l % 16, dims 32 kk + 8 (l / 16) ..
    __device__ __forceinline__ gqa_u4 s_frag(const gqa_u4* tile, int hf, int kk) const {
        if constexpr (kXor)
            return *reinterpret_cast<const gqa_u4*>(reinterpret_cast<const char*>(tile + 16 * hf * CPR) + (s_at ^ (kk << 6)));
        else return tile_s_frag<CPR>(tile, lane, hf, kk);
    }
    // rows 16 h + 4 (l / 16) .. + 3 of dim 16 dt + l % 16
    __device__ __forceinline__ uint2 tr_half(const gqa_u4* tile, int h, int dt) const {
        const char* p = reinterpret_cast<const char*>(tile + 16 * h * CPR) +
                        (kXor ? t_at ^ (dt << 5) : lane.t_off[dt & 1][0] + 64 * (dt >> 1));
        return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) gqa_v4s*)(p)));
    }
};

template <typename T, int HD, bool KCTX>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
paged_items_kernel(BatchArgs<T> a) {
    constexpr int KK = HD / 32, DT = HD / 16, CPR = HD / 8, NS = pb_stages<HD>(), GPW = CPR / 4, R = kPbTile;
    // a stage per array, so that a wait for one stage's loads never covers another's reads
    __shared__ __align__(16) gqa_u4 K0[R * CPR], V0[R * CPR], K1[R * CPR], V1[R * CPR];
    __shared__ __align__(16) gqa_u4 K2[NS == 3 ? R * CPR : 1], V2[NS == 3 ? R * CPR : 1];
    __shared__ PbEnd end;
    using M = Mfma16<T>;
    const PbWork w = pb_work(a);
    if (!w.any) return;
    const PbItem& s = w.s;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int lr = lane & 15, lq = lane >> 4;
    const PbLane<CPR> tl(lq, lr);
    const int kend = min(s.key1, s.key0 + s.tile1 * R);
    const int32_t* trow = a.table + (int64_t)s.row * a.table_ld;

    // pages of this wave's quarter of the tiles jb .. jb + 63, one per lane
    int jb = s.tile0, pgv;
    auto pages = [&]() {
        const int64_t t = (int64_t)s.key0 + (int64_t)(jb + lane) * R + 16 * wave;
        pgv = trow[min(t, (int64_t)a.cap - 1) >> a.log_ps];
    };
    pages();
    const bool odd_mine = pb_odd(a, s);
    uint32_t voff[GPW];
#pragma unroll
    for (int j = 0; j < GPW; ++j) {
        const int p = 64 * j + lane, row = p / CPR, c = p - row * CPR;
        voff[j] = (uint32_t)(row * (int)a.ps_tok * (int)sizeof(T)) + (uint32_t)(c ^ tl.swz(row)) * 16u;
    }
    auto kst = [&](auto s_) -> gqa_u4* {
        constexpr int I = decltype(s_)::value;
        return I == 0 ? K0 : I == 1 ? K1 : K2;
    };
    auto vst = [&](auto s_) -> gqa_u4* {
        constexpr int I = decltype(s_)::value;
        return I == 0 ? V0 : I == 1 ? V1 : V2;
    };
    // this wave's quarter of tile j, 2 GPW loads (past the item's end: zeros)
    auto load_tile = [&](auto s_, int j) {
        const int t = s.key0 + j * R + 16 * wave;
        const int rows = j < s.tile1 ? min(16, kend - t) : 0;
        int bytes = 0;
        int64_t off = 0;
        if (rows > 0) {
            if (j - jb >= 64) {
                jb += 64;
                pages();
            }
            const int page = __builtin_amdgcn_readlane(pgv, j - jb);
            if ((unsigned)page < (unsigned)a.n_pages) {          // (all are, unless the table changed since the plan)
                bytes = ((rows - 1) * (int)a.ps_tok + HD) * (int)sizeof(T);
                off = (int64_t)page * a.ps_page + (int64_t)(t & ((1 << a.log_ps) - 1)) * a.ps_tok + w.kvh * a.ps_head;
            }
        }
        const auto rk = __builtin_amdgcn_make_buffer_rsrc((void*)(a.kp + off), (short)0, bytes, kBufferDword3);
        const auto rv = __builtin_amdgcn_make_buffer_rsrc((void*)(a.vp + off), (short)0, bytes, kBufferDword3);
#pragma unroll
        for (int i = 0; i < GPW; ++i) {
            dma16(rk, kst(s_) + 64 * (wave * GPW + i), voff[i], 0);
            dma16(rv, vst(s_) + 64 * (wave * GPW + i), voff[i], 0);
        }
    };
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I4 = std::integral_constant<int, 4>;
    const bool odd = __syncthreads_or(odd_mine);

    auto body = [&](auto kw_, auto nq_) __attribute__((always_inline)) {
        constexpr int KW = decltype(kw_)::value, NQ = decltype(nq_)::value, QW = 4 / KW;
        constexpr int NHF = KW == 4 ? 1 : 2;                 // 16-row parts of a fold
        constexpr int FOLDS = 4 / (KW * NHF);                // folds of a wave per tile
        const int kg = wave / QW, x0 = (wave & (QW - 1)) * 16 * NQ;
        // q of column lr, positions that the column sees; (columns without a query: the last one's)
        uint4 qf[NQ][KK];
        int sees[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const int x = min(x0 + 16 * n + lr, s.nq - 1);
            const T* q = a.q_out + ((int64_t)pb_token(a, s, x) * a.QH + w.kvh * a.G + (s.x0 + x) % a.G) * HD + 8 * lq;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) qf[n][kk] = *reinterpret_cast<const uint4*>(q + 32 * kk);
            sees[n] = min(pb_sees(a, s, x), kend);
        }
        const int sees_first = __builtin_amdgcn_readfirstlane(min(pb_sees(a, s, min(x0, s.nq - 1)), kend));
        const int seen_by_all = pb_sees(a, s, 0);            // positions that every query of the block sees
        float mh[NQ], off[NQ], lh[NQ];                       // the reference, minus it (0 before there is one), the sum
        pg_f32x4 accC[NQ][DT], accK[NQ][KCTX ? DT : 1];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            mh[n] = -INFINITY;
            off[n] = lh[n] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) accC[n][dt] = pg_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int dt = 0; dt < (KCTX ? DT : 1); ++dt) accK[n][dt] = pg_f32x4{0.f, 0.f, 0.f, 0.f};
        }
        // rows r0 .. of the stage at tk, tv; the last `dirty` of the block's rows here are not seen by all its queries
        auto fold = [&](const gqa_u4* tk, const gqa_u4* tv, int r0, int dirty) __attribute__((always_inline)) {
            pg_f32x4 sc[NQ][NHF];
#pragma unroll
            for (int hf = 0; hf < NHF; ++hf) {
#pragma unroll
                for (int n = 0; n < NQ; ++n) sc[n][hf] = pg_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    const uint4 f = __builtin_bit_cast(uint4, tl.s_frag(tk, hf, kk));
#pragma unroll
                    for (int n = 0; n < NQ; ++n) sc[n][hf] = M::dot(f, qf[n][kk], sc[n][hf]);
                }
            }
            if (dirty > 0) {                         // the block's rows of this fold, now that all waves have their scores
                lds_barrier();
                gqa_u4* const k = const_cast<gqa_u4*>(tk - (KW == 1 ? 0 : kg * (R / KW) * CPR));
                gqa_u4* const v = const_cast<gqa_u4*>(tv - (KW == 1 ? 0 : kg * (R / KW) * CPR));
                constexpr int rows = KW == 1 ? 16 * NHF : R;
                for (int i = max(rows - dirty, 0) * CPR + tid; i < rows * CPR; i += 256) {
                    k[i] = pb_finite<T>(k[i]);
                    v[i] = pb_finite<T>(v[i]);
                }
                lds_barrier();
            }
            const bool mask = r0 + 16 * NHF > sees_first;        // wave-uniform
            if (mask) {
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int hf = 0; hf < NHF; ++hf)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (r0 + 16 * hf + 4 * lq + r >= sees[n]) sc[n][hf][r] = -INFINITY;
            }
            float mx[NQ];
            bool rise = false;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                mx[n] = -INFINITY;
#pragma unroll
                for (int hf = 0; hf < NHF; ++hf)
#pragma unroll
                    for (int r = 0; r < 4; ++r) mx[n] = fmaxf(mx[n], sc[n][hf][r]);
                mx[n] = fmaf(mx[n], a.qscale, -M::kShift);
                rise |= mx[n] > mh[n] + M::kLag;
            }
            if (__any(rise)) {
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const float mnew = raised(mh[n], max_16_32(mx[n]), M::kLag);
                    const float corr = mnew == mh[n] ? 1.0f : __builtin_amdgcn_exp2f(mh[n] - mnew);
                    const bool first = mh[n] == -INFINITY;       // the sums are zero
                    mh[n] = mnew;
                    off[n] = mnew == -INFINITY ? 0.0f : -mnew;   // (nothing seen yet: e^-inf, not e^NaN)
                    lh[n] *= corr;
                    if (__any(!first && corr != 1.0f)) {
                        pg_f32x4 cf;
#pragma unroll
                        for (int r = 0; r < 4; ++r) cf[r] = __shfl(first ? 1.0f : corr, 4 * lq + r, 64);
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) {
                            accC[n][dt] *= cf;
                            if constexpr (KCTX) accK[n][dt] *= cf;
                        }
                    }
                }
            }
            float pv[NQ][NHF][4];
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
#pragma unroll
                for (int hf = 0; hf < NHF; ++hf)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        pv[n][hf][r] = __builtin_amdgcn_exp2f(fmaf(sc[n][hf][r], a.qscale, off[n]));
                        lh[n] += pv[n][hf][r];
                    }
            }
            // the weights enter the products rounded to the storage type (half a step of
            // it, relative, per weight, down to Mfma16's smallest: below the rounding of
            // the outputs); their sum l is that of the unrounded ones
            uint4 pa[NQ];
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                pa[n] = make_uint4(M::pack(pv[n][0][0], pv[n][0][1]), M::pack(pv[n][0][2], pv[n][0][3]), 0, 0);
                if constexpr (NHF > 1) {
                    pa[n].z = M::pack(pv[n][1][0], pv[n][1][1]);
                    pa[n].w = M::pack(pv[n][1][2], pv[n][1][3]);
                }
            }
            auto frag = [&](const gqa_u4* tile, int dt) __attribute__((always_inline)) {
                const uint2 lo = tl.tr_half(tile, 0, dt);
                uint2 hi = make_uint2(0, 0);         // (of 16 rows the other half meets zero weights)
                if constexpr (NHF > 1) hi = tl.tr_half(tile, 1, dt);
                return make_uint4(lo.x, lo.y, hi.x, hi.y);
            };
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const uint4 fv = frag(tv, dt);
#pragma unroll
                for (int n = 0; n < NQ; ++n) accC[n][dt] = M::dot(pa[n], fv, accC[n][dt]);
                if constexpr (KCTX) {
                    const uint4 fk = frag(tk, dt);
#pragma unroll
                    for (int n = 0; n < NQ; ++n) accK[n][dt] = M::dot(pa[n], fk, accK[n][dt]);
                }
            }
            __builtin_amdgcn_s_setprio(0);
        };
        // a step computes tile j from its stage, requests tile j + NS - 1 into the stage that every
        // wave is done with, waits for tile j + 1 and passes one barrier
        auto step = [&](auto s_, int j) __attribute__((always_inline)) {
            constexpr int cur = decltype(s_)::value;
            load_tile(std::integral_constant<int, (cur + NS - 1) % NS>{}, j + NS - 1);
#pragma unroll
            for (int u = 0; u < FOLDS; ++u) {
                const int row = kg * (R / KW) + u * 16 * NHF, r0 = s.key0 + j * R + row;
                // (unconditionally: a branch around it costs the loop's registers more than what a wave
                // without a query, or that sees nothing here yet, could save)
                // (the block's: rows of the fold where all waves have the same, else of the tile)
                const int end = KW == 1 ? r0 + 16 * NHF : s.key0 + (j + 1) * R;
                fold(kst(s_) + row * CPR, vst(s_) + row * CPR, r0, odd ? end - seen_by_all : 0);
            }
            wait_vmcnt<2 * GPW * (NS - 2)>();
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        };
        load_tile(std::integral_constant<int, 0>{}, s.tile0);
        if constexpr (NS == 3) load_tile(I1{}, s.tile0 + 1);
        wait_vmcnt<2 * GPW * (NS - 2)>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
                asm volatile("" : "+v"(qf[n][kk].x), "+v"(qf[n][kk].y), "+v"(qf[n][kk].z), "+v"(qf[n][kk].w));
        for (int j = s.tile0;; j += NS) {         // (an item has a tile)
            step(std::integral_constant<int, 0>{}, j);
            if (j + 1 >= s.tile1) break;
            step(I1{}, j + 1);
            if (j + 2 >= s.tile1) break;
            if constexpr (NS == 3) {
                step(I2{}, j + 2);
                if (j + 3 >= s.tile1) break;
            }
        }
        wait_vmcnt<0>();                             // no load into LDS outlives the loop
        // wave w's sums in the w-th of four stage arrays, whose size they have
        static_assert(16 * 2 * HD * sizeof(float) == sizeof(K0), "a wave's sums of 16 queries fill a stage");
        auto part = [&](int i) { return reinterpret_cast<float*>(i == 0 ? K0 : i == 1 ? V0 : i == 2 ? K1 : V1); };
        // records of queries that one wave has alone go out of its registers as they are
        if (KW == 1 && s.rec >= 0 && !odd) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const int x = 16 * (NQ * wave + n);
                const int64_t to = w.kvh * a.at.cap_recs + s.rec + x;
                lh[n] = sum_16_32(lh[n]);
                if (lq == 0 && x + lr < s.nq) *reinterpret_cast<float2*>(a.rec + a.rec_ml + 2 * (to + lr)) = make_float2(mh[n], lh[n]);
                float* rec = a.rec + (to + 4 * lq) * 2 * HD + lr;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (x + 4 * lq + i >= s.nq) break;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        rec[i * 2 * HD + 16 * dt] = accC[n][dt][i];
                        if constexpr (KCTX) rec[i * 2 * HD + HD + 16 * dt] = accK[n][dt][i];
                    }
                }
            }
            return;
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            __syncthreads();                         // the stages, or the last queries' sums, are read
            lh[n] = sum_16_32(lh[n]);
            if (lq == 0) end.ml[wave][lr] = make_float2(mh[n], lh[n]);
            pg_f32x4* mine = reinterpret_cast<pg_f32x4*>(part(wave)) + lane;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                mine[64 * dt] = accC[n][dt];
                if constexpr (KCTX) mine[64 * (DT + dt)] = accK[n][dt];
            }
            pb_finish<HD, KCTX, QW>(a, w, 16 * n, 16 * NQ, odd, end, part);
        }
    };
    if (s.nq <= 16) body(I4{}, I1{});
    else if (s.nq <= 32) body(I2{}, I1{});
    else if (s.nq <= 64) body(I2{}, I2{});
    else body(I1{}, I2{});
}

// ------------------------------------------------------------------ fp32 form
// fp32 (whose products stay in fp32, on v_mfma_f32_16x16x4) and the head sizes the form
// above does not take, converted to fp32 as they are staged.  The same waves and query
// blocks; RT positions per step in one LDS buffer, the next ones in flight in registers.
// The products' operands may take the dimensions in any order that both share: lane
// group lq takes HD / 4 neighbouring ones of them, so that a lane's are 16-byte reads.
// Three prompts to 257 tokens 14.1 us, 4 rows to 1300 9.5: the chain item, page, tile, sums.  Long prompts
// by the operands of the products, of which each is one 4-byte LDS read that no second query block
// shares (4 x 1024 tokens behind 500 322 us, 59 TFLOP/s of 154).  16-bit heads pay the fp32 products'
// rate: 4 x 1024 tokens behind 500 with 8 heads of 256 662 us, 62 rows behind 16384 with 32 of
// them 743 (of 128 on the 16-bit products 52), 32 x 128 tokens behind 1920 with 8 heads of 16 114.
template <typename T, int HD, bool KCTX>
__global__ void __launch_bounds__(256)
paged_items_f32_kernel(BatchArgs<T> a) {
    constexpr int HDP = HD < 16 ? 16 : HD;           // heads of 8 are filled up with zeros
    constexpr int RT = HDP <= 128 ? 64 : 32, PITCH = HDP + 4, Q4 = HDP / 16, DT = HDP / 16;
    constexpr int EP = 16 / sizeof(T), PR = HD / EP; // elements of a 16-byte piece, pieces of a row
    constexpr int NP = (RT * PR + 255) / 256;        // pieces per thread and tensor
    constexpr int kTile = 2 * RT * PITCH, kRed = 4 * 16 * 2 * HDP;
    __shared__ __align__(16) float lds[kTile > kRed ? kTile : kRed];
    __shared__ PbEnd end;
    const PbWork w = pb_work(a);
    if (!w.any) return;
    const PbItem& s = w.s;
    // 64 of the segment's queries, 32 where that leaves blocks too few: blocks of other y take
    // the others (when it was taken, 64 / 32 queries: 4 x 1024 new tokens 324 / 362 us, 3 of 1 to 257 25.8 / 19.0)
    const int per = a.plan[1] >= a.at.slots ? 64 : 32, xb = per * blockIdx.y, nq = min(s.nq - xb, per);
    if (nq <= 0) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int lr = lane & 15, lq = lane >> 4;
    const int QW = nq <= 16 ? 1 : nq <= 32 ? 2 : 4, KW = 4 / QW;
    const int x0 = xb + 16 * (wave & (QW - 1)), kg = wave / QW;
    const int k0 = s.key0 + s.tile0 * kPbTile, kend = min(s.key1, s.key0 + s.tile1 * kPbTile);
    const int32_t* trow = a.table + (int64_t)s.row * a.table_ld;
    const int ps_mask = (1 << a.log_ps) - 1;
    float* const tk = lds;
    float* const tv = lds + RT * PITCH;
    if constexpr (HDP > HD) {
        for (int i = tid; i < kTile; i += 256) lds[i] = 0.0f;
        __syncthreads();
    }
    // pages of 64 runs of 16 positions from jb on, one per lane
    int jb = k0, pgv;
    auto pages = [&]() { pgv = trow[min((int64_t)jb + 16 * lane, (int64_t)a.cap - 1) >> a.log_ps]; };
    pages();
    const int xq = min(x0 + lr, s.nq - 1);
    const bool odd_mine = pb_odd(a, s);
    // q of column lr, dimensions lq HDP / 4 ..
    float qf[HDP / 4];
    {
        const T* q = a.q_out + ((int64_t)pb_token(a, s, xq) * a.QH + w.kvh * a.G + (s.x0 + xq) % a.G) * HD;
#pragma unroll
        for (int i = 0; i < HDP / 4; ++i) {
            const int d = lq * (HDP / 4) + i;
            qf[i] = d < HD ? ld(q + d) : 0.0f;
        }
    }
    const int sees = min(pb_sees(a, s, xq), kend);
    const int sees_first = __builtin_amdgcn_readfirstlane(min(pb_sees(a, s, min(x0, s.nq - 1)), kend));
    const int seen_by_all = pb_sees(a, s, 0);        // positions that every query of the block sees
    const int sees_last = x0 >= s.nq ? 0 : __builtin_amdgcn_readfirstlane(min(pb_sees(a, s, min(x0 + 15, s.nq - 1)), kend));
    u32x4 kr[NP], vr[NP];
    auto load = [&](int t0) {                        // positions t0 .. t0 + RT - 1
        if (t0 < kend && t0 - jb >= 16 * 64) {
            jb += 16 * 64;
            pages();
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = i * 256 + tid, row = p / PR, c = p - row * PR, t = t0 + row;
            const int page = __shfl(pgv, ((t - jb) >> 4) & 63, 64);
            kr[i] = vr[i] = u32x4{0, 0, 0, 0};
            if (row < RT && t < kend && (unsigned)page < (unsigned)a.n_pages) {
                const int64_t off = (int64_t)page * a.ps_page + (int64_t)(t & ps_mask) * a.ps_tok + w.kvh * a.ps_head + c * EP;
                kr[i] = *reinterpret_cast<const u32x4*>(a.kp + off);
                vr[i] = *reinterpret_cast<const u32x4*>(a.vp + off);
            }
        }
    };
    auto put = [&](float* at, u32x4 v) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<u32x4*>(at) = v;
        } else {
            float f[8];
            Vec8<T>::load(reinterpret_cast<const T*>(&v), f);
            Vec8<float>::store(at, f);
        }
    };
    const bool odd = __syncthreads_or(odd_mine);
    float mh = -INFINITY, off = 0.0f, lh = 0.0f;
    pg_f32x4 accC[DT], accK[KCTX ? DT : 1];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) accC[dt] = pg_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < (KCTX ? DT : 1); ++dt) accK[dt] = pg_f32x4{0.f, 0.f, 0.f, 0.f};
    load(k0);
    for (int t0 = k0; t0 < kend; t0 += RT) {
        __syncthreads();                             // the tile's last reads
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = i * 256 + tid, row = p / PR, c = p - row * PR;
            if (row < RT) {
                put(tk + row * PITCH + c * EP, kr[i]);
                put(tv + row * PITCH + c * EP, vr[i]);
            }
        }
        load(t0 + RT);
        lds_barrier();
        for (int hf = kg; hf < RT / 16; hf += KW) {
            const int r0 = t0 + 16 * hf;
            if (r0 >= sees_last) break;              // (a wave's: uniform; at once where it has no query)
            // four sums side by side: a product waits for the one before it in its sum
            pg_f32x4 part[4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            const float* kq = tk + (16 * hf + lr) * PITCH + lq * (HDP / 4);
#pragma unroll
            for (int i = 0; i < Q4; ++i) {
                const pg_f32x4 kx = *reinterpret_cast<const pg_f32x4*>(kq + 4 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) part[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[e], qf[4 * i + e], part[e], 0, 0, 0);
            }
            pg_f32x4 sc = (part[0] + part[1]) + (part[2] + part[3]);
            const bool mask = r0 + 16 > sees_first;
            float mx = -INFINITY, pv[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (mask && r0 + 4 * lq + r >= sees) sc[r] = -INFINITY;
                mx = fmaxf(mx, sc[r]);
            }
            mx *= a.qscale;
            if (__any(mx > mh + kPgLag)) {
                const float mnew = raised(mh, max_16_32(mx));
                const float corr = mnew == mh ? 1.0f : __builtin_amdgcn_exp2f(mh - mnew);
                const bool first = mh == -INFINITY;              // the sums are zero
                mh = mnew;
                off = mnew == -INFINITY ? 0.0f : -mnew;
                lh *= corr;
                pg_f32x4 cf;
#pragma unroll
                for (int r = 0; r < 4; ++r) cf[r] = __shfl(first ? 1.0f : corr, 4 * lq + r, 64);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    accC[dt] *= cf;
                    if constexpr (KCTX) accK[dt] *= cf;
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                pv[r] = __builtin_amdgcn_exp2f(fmaf(sc[r], a.qscale, off));
                lh += pv[r];
            }
            const bool dirty = odd && r0 + 16 > seen_by_all;     // rows that not all queries see (pb_odd)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * hf + 4 * lq + r;
                float v[DT], k[DT];
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    v[dt] = tv[row * PITCH + lr + 16 * dt];
                    if constexpr (KCTX) k[dt] = tk[row * PITCH + lr + 16 * dt];
                }
                if (dirty) {
                    const bool partly = t0 + row >= seen_by_all;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        if (partly && !(fabsf(v[dt]) < INFINITY)) v[dt] = 0.0f;
                        if (KCTX && partly && !(fabsf(k[dt]) < INFINITY)) k[dt] = 0.0f;
                    }
                }
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    accC[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(pv[r], v[dt], accC[dt], 0, 0, 0);
                    if constexpr (KCTX) accK[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(pv[r], k[dt], accK[dt], 0, 0, 0);
                }
            }
        }
    }
    lh = sum_16_32(lh);
    __syncthreads();
    auto part = [&](int i) { return lds + i * 16 * 2 * HDP; };
    if (lq == 0) end.ml[wave][lr] = make_float2(mh, lh);
    pg_f32x4* mine = reinterpret_cast<pg_f32x4*>(part(wave)) + lane;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        mine[64 * dt] = accC[dt];
        if constexpr (KCTX) mine[64 * (DT + dt)] = accK[dt];
    }
    if (QW == 4) pb_finish<HDP, KCTX, 4>(a, w, xb, 16, odd, end, part);
    else if (QW == 2) pb_finish<HDP, KCTX, 2>(a, w, xb, 16, odd, end, part);
    else pb_finish<HDP, KCTX, 1>(a, w, xb, 16, odd, end, part);
}

// ------------------------------------------------------------------ the join
// The queries whose sums are in records, those of their own segment's chunks and of the
// group's segment that holds them.  Of few records (kPbFew) a block's four waves take a
// query each, all its records in flight; of more it takes one query: wave w records w,
// w + 4, .., kPbJoin of them in flight, and the waves meet in LDS.  Bound by the chain count,
// task, records where those are few (32 rows behind 2048 4.0 us), by the records' bytes else (62
// rows behind 16384, 32 heads of 128: 10.3 us).  Without Kctx that half of a record is neither
// written nor used, but it is read (10.5).
constexpr int kPbJoin = 8;

// What a part's sums weigh beside those of a part with the greater reference `most`.  Never
// zero: an infinity that an item's end has put into a part stays one.  (2^-80 of a part's l, which is below
// 2^40, is less than 2^-40 of the sum, whose l is at least 1: nothing of what is finite.)
__device__ __forceinline__ float pb_weight(float m, float most) {
    return most == -INFINITY ? 1.0f : fmaxf(__builtin_amdgcn_exp2f(m - most), 0x1p-80f);
}

// (m, l, v) and a record's (e, y) as one
template <int NV>
__device__ __forceinline__ void pb_add(float& m, float& l, pg_f32x4 (&v)[NV], float2 e, const pg_f32x4 (&y)[NV]) {
    const float most = fmaxf(m, e.x);
    const float f = pb_weight(m, most), g = pb_weight(e.x, most);
    l = fmaf(l, f, e.y * g);
#pragma unroll
    for (int k = 0; k < NV; ++k) v[k] = v[k] * f + y[k] * g;
    m = most;
}

template <typename T, int HD>
__global__ void __launch_bounds__(256)
paged_batch_join_kernel(BatchArgs<T> a) {
    constexpr int HDP = HD < 16 ? 16 : HD;
    constexpr int NV = HDP > 128 ? 2 : 1, NL = HDP / 2 / NV;   // lanes of four sums
    __shared__ float2 ml[4];
    __shared__ __align__(16) float sums[4][2 * HDP];
    const int kvh = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int at = min(lane, NL - 1);
    const bool kctx = a.k_out != nullptr;
    const PbJoin* joins = reinterpret_cast<const PbJoin*>(a.plan + a.at.joins);
    int next = a.plan[a.at.tasks + min((int)blockIdx.x, a.at.cap_tasks - 1)];    // with the count that says whether it is one
    const int n_tasks = min(a.plan[2], a.at.cap_tasks);
    if (!plan_fits(a)) return;
    const float* rec = a.rec + kvh * a.at.cap_recs * 2 * HDP;
    const float* rml = a.rec + a.rec_ml + kvh * a.at.cap_recs * 2;
    for (int task = blockIdx.x; task < n_tasks; task += gridDim.x) {
        if (task != (int)blockIdx.x) next = a.plan[a.at.tasks + task];
        const PbJoin t = joins[next / kPbQ];
        const int y = next % kPbQ, nx = min(4, t.nq - y);
        const int base = t.base, x0 = t.x0 + y, own = t.own + y, own_step = t.nq, nc = t.common_n, n = nc + t.own_n;
        // the group's segments: 128 queries each but the last, all of the same chunks; query
        // `cut` of the four is the first of the next one
        const int g = t.g0 + y, seg = g / kPbQ, r0 = t.common0 + seg * kPbQ * nc, cut = (seg + 1) * kPbQ - g;
        const int step0 = min(kPbQ, t.group_q - seg * kPbQ), common0 = r0 + g - seg * kPbQ;
        const int step1 = min(kPbQ, t.group_q - (seg + 1) * kPbQ), common1 = r0 + kPbQ * nc + g - (seg + 1) * kPbQ;
        // record c of query i
        auto place = [=](int i, int c) __attribute__((always_inline)) -> int64_t {
            const int c0 = common0 + c * step0, c1 = common1 + c * step1, c2 = own + (c - nc) * own_step;
            return (c >= nc ? c2 : i < cut ? c0 : c1) + i;
        };
        auto out = [=](int i, int d2, const float (&o)[4]) __attribute__((always_inline)) {   // four sums of query i from d2 on
            const int which = d2 >= HDP, d = d2 - which * HDP;
            if ((which && !kctx) || (HDP > HD && d >= HD)) return;
            const int x = x0 + i, h = kvh * a.G + x % a.G;
            store_e<T, 4>((which ? a.k_out : a.c_out) + (int64_t)(base + x / a.G) * a.out_ld + (int64_t)h * HD + d, o);
        };
        if (n <= kPbFew) {
            const int i = wave;
            if (i >= nx) continue;
            float2 e[kPbFew];
            pg_f32x4 y[kPbFew][NV];
#pragma unroll
            for (int c = 0; c < kPbFew; ++c) {
                const int64_t r = place(i, min(c, n - 1));
                e[c] = *reinterpret_cast<const float2*>(rml + 2 * r);
#pragma unroll
                for (int v = 0; v < NV; ++v)
                    y[c][v] = *reinterpret_cast<const pg_f32x4*>(rec + r * 2 * HDP + 4 * (at + NL * v));
            }
            float m = e[0].x, l = e[0].y;
#pragma unroll
            for (int c = 1; c < kPbFew; ++c)
                if (c < n) pb_add<NV>(m, l, y[0], e[c], y[c]);
            const float inv = 1.0f / l;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const float o[4] = {y[0][v][0] * inv, y[0][v][1] * inv, y[0][v][2] * inv, y[0][v][3] * inv};
                if (lane < NL) out(i, 4 * (lane + NL * v), o);
            }
            continue;
        }
        float m = -INFINITY, l = 0.0f;
        pg_f32x4 sum[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) sum[v] = pg_f32x4{0.f, 0.f, 0.f, 0.f};
        for (int c0 = wave; c0 < n; c0 += 4 * kPbJoin) {
            float2 e[kPbJoin];
            pg_f32x4 z[kPbJoin][NV];
#pragma unroll
            for (int k = 0; k < kPbJoin; ++k) {
                const int64_t r = place(0, min(c0 + 4 * k, n - 1));
                e[k] = *reinterpret_cast<const float2*>(rml + 2 * r);
#pragma unroll
                for (int v = 0; v < NV; ++v) z[k][v] = *reinterpret_cast<const pg_f32x4*>(rec + r * 2 * HDP + 4 * (at + NL * v));
            }
#pragma unroll
            for (int k = 0; k < kPbJoin; ++k)
                if (c0 + 4 * k < n) pb_add<NV>(m, l, sum, e[k], z[k]);
        }
        __syncthreads();                             // the last task's sums are read
        if (lane == 0) ml[wave] = make_float2(m, l);
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (lane < NL) *reinterpret_cast<pg_f32x4*>(&sums[wave][4 * (lane + NL * v)]) = sum[v];
        __syncthreads();
        for (int k = threadIdx.x; k < HDP / 2; k += 256) {
            const int d2 = 4 * k;
            float most = -INFINITY, all = 0.0f;
#pragma unroll
            for (int v = 0; v < 4; ++v) most = fmaxf(most, ml[v].x);
            float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float f = pb_weight(ml[v].x, most);
                all = fmaf(ml[v].y, f, all);
#pragma unroll
                for (int q = 0; q < 4; ++q) o[q] = fmaf(sums[v][d2 + q], f, o[q]);
            }
            const float inv = 1.0f / all;
#pragma unroll
            for (int q = 0; q < 4; ++q) o[q] *= inv;
            out(0, d2, o);
        }
    }
}

// ------------------------------------------------------------------ host side

static int batch_sizes(const char* who, int64_t R, int64_t N, int64_t QH, int64_t KVH, int64_t NP, int64_t PS, int64_t MP,
                       int64_t table_ld) {
    LOOM_CHECK(R >= 0 && R <= kPbMaxRows, "%s: 0 to %d rows, got %lld", who, kPbMaxRows, (long long)R);
    LOOM_CHECK(N >= 0 && N <= kPbMaxTokens, "%s: 0 to %lld tokens, got %lld", who, (long long)kPbMaxTokens, (long long)N);
    LOOM_CHECK(KVH >= 1 && QH >= KVH && QH <= 1024 && QH % KVH == 0, "%s: bad heads QH=%lld KVH=%lld", who,
               (long long)QH, (long long)KVH);
    LOOM_CHECK(PS >= 16 && PS <= 1024 && (PS & (PS - 1)) == 0, "%s: page_size must be a power of two from 16 to 1024, got %lld",
               who, (long long)PS);
    LOOM_CHECK(NP >= 1 && NP < ((int64_t)1 << 30), "%s: bad n_pages %lld", who, (long long)NP);
    LOOM_CHECK(MP >= 1 && MP <= ((int64_t)1 << 24) / PS && table_ld >= MP,
               "%s: the table must hold 1 page to 2^24 tokens per row (max_pages=%lld, row stride %lld)", who,
               (long long)MP, (long long)table_ld);
    return LOOM_OK;
}

struct BatchCall {
    const void* qkv;
    int64_t qkv_ld;
    void *kp, *vp;
    int64_t page_stride, token_stride, head_stride, n_pages, page_size;
    const int32_t* table;
    int64_t table_ld, max_pages, rows;
    const int32_t *rows_of, *positions;
    const int64_t* slots;
    const void* plan;
    int64_t plan_bytes;
    const float *cosv, *sinv;
    int64_t n_pos;
    void *q_out, *c_out, *k_out;
    int64_t out_ld;
    void* ws;
    int64_t ws_bytes, N, QH, KVH, HD;
};

static int64_t pb_rec_floats(const PbLayout& at, int64_t KVH, int64_t HD) {
    const int64_t HDP = HD < 16 ? 16 : HD;
    return KVH * at.cap_recs * (2 * HDP + 2);
}

template <typename T>
static int batch_launch(const BatchCall& c, hipStream_t st) {
    BatchArgs<T> a{};
    a.qkv = (const T*)c.qkv;
    a.qkv_ld = c.qkv_ld;
    a.kp = (T*)c.kp;
    a.vp = (T*)c.vp;
    a.ps_page = c.page_stride;
    a.ps_tok = c.token_stride;
    a.ps_head = c.head_stride;
    a.table = c.table;
    a.table_ld = c.table_ld;
    a.positions = c.positions;
    a.rows_of = c.rows_of;
    a.slots_of = c.slots;
    a.cosv = c.cosv;
    a.sinv = c.sinv;
    a.q_out = (T*)c.q_out;
    a.c_out = (T*)c.c_out;
    a.k_out = (T*)c.k_out;
    a.out_ld = c.out_ld;
    a.plan = (const int32_t*)c.plan;
    a.at = pb_layout(c.rows, c.N, c.QH, c.KVH);
    a.rec = (float*)c.ws;
    const int64_t HDP = c.HD < 16 ? 16 : c.HD;
    a.rec_ml = c.KVH * a.at.cap_recs * 2 * HDP;
    a.odd = (uint8_t*)((float*)c.ws + pb_rec_floats(a.at, c.KVH, c.HD));
    a.R = (int)c.rows;
    a.N = (int)c.N;
    a.QH = (int)c.QH;
    a.KVH = (int)c.KVH;
    a.G = (int)(c.QH / c.KVH);
    a.HD = (int)c.HD;
    a.log_ps = __builtin_ctzll((unsigned long long)c.page_size);
    a.cap = (int)(c.max_pages * c.page_size);
    a.n_pages = (int)c.n_pages;
    a.n_pos = (int)min(c.n_pos, (int64_t)1 << 30);
    a.qscale = kLog2e / sqrtf((float)c.HD);
    const dim3 appends((unsigned)c.N);
    if (c.HD >= 16) hipLaunchKernelGGL((paged_append_kernel<T, 8>), appends, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_append_kernel<T, 4>), appends, dim3(256), 0, st, a);
    if (int rc = launch_status("loom_paged_batch_step(append)")) return rc;
    // no more items than there are segments times a row's tiles (fp32, 3 rows
    // of up to 257: 15.5 -> 13.8 us without the blocks that can have nothing)
    const int64_t most = (int64_t)(a.at.cap_items - a.at.slots) * ceil_div((int64_t)a.cap, kPbTile);
    const dim3 grid((unsigned)((most < a.at.cap_items ? most : a.at.cap_items) * c.KVH));
    bool done = false;
    if constexpr (sizeof(T) == 2) {
#define LOOM_PB_M(HDV)                                                                              \
        if (c.HD == HDV) {                                                                          \
            if (c.k_out) hipLaunchKernelGGL((paged_items_kernel<T, HDV, true>), grid, dim3(256), 0, st, a); \
            else hipLaunchKernelGGL((paged_items_kernel<T, HDV, false>), grid, dim3(256), 0, st, a); \
            done = true;                                                                            \
        }
        LOOM_PB_M(96) LOOM_PB_M(128) LOOM_PB_M(64) LOOM_PB_M(32)
#undef LOOM_PB_M
#define LOOM_PB_F(HDV)                                                                              \
        if (c.HD == HDV) {                                                                          \
            const dim3 halves(grid.x, kPbQ / 32);                                                   \
            if (c.k_out) hipLaunchKernelGGL((paged_items_f32_kernel<T, HDV, true>), halves, dim3(256), 0, st, a); \
            else hipLaunchKernelGGL((paged_items_f32_kernel<T, HDV, false>), halves, dim3(256), 0, st, a); \
            done = true;                                                                            \
        }
        LOOM_PB_F(8) LOOM_PB_F(16) LOOM_PB_F(256)
    } else {
        LOOM_PB_F(96) LOOM_PB_F(128) LOOM_PB_F(64) LOOM_PB_F(32) LOOM_PB_F(16) LOOM_PB_F(8) LOOM_PB_F(256)
#undef LOOM_PB_F
    }
    LOOM_CHECK(done, "paged_batch_step: unsupported head_dim %lld (8, 16, 32, 64, 96, 128 or 256)", (long long)c.HD);
    if (int rc = launch_status("loom_paged_batch_step(items)")) return rc;
    // (4096 blocks instead: 4.9 us for 4.4 of few joins, 7.9 for 7.4 of many)
    const int64_t joins = ceil_div(1024, c.KVH);
    const dim3 jgrid((unsigned)(joins < a.at.cap_tasks ? joins : a.at.cap_tasks), (unsigned)c.KVH);
#define LOOM_PB_J(HDV)                                                                              \
    if (c.HD == HDV) hipLaunchKernelGGL((paged_batch_join_kernel<T, HDV>), jgrid, dim3(256), 0, st, a);
    LOOM_PB_J(96) LOOM_PB_J(128) LOOM_PB_J(64) LOOM_PB_J(32) LOOM_PB_J(16) LOOM_PB_J(8) LOOM_PB_J(256)
#undef LOOM_PB_J
    return launch_status("loom_paged_batch_step(join)");
}

}  // namespace loom

using namespace loom;

extern "C" int64_t loom_paged_plan_bytes(int64_t rows, int64_t n_tokens, int64_t QH, int64_t KVH) {
    if (rows < 0 || rows > kPbMaxRows || n_tokens < 0 || n_tokens > kPbMaxTokens || KVH < 1 || QH < KVH || QH > 1024 || QH % KVH != 0)
        return 0;
    return pb_layout(rows, n_tokens, QH, KVH).total * (int64_t)sizeof(int32_t);
}

extern "C" int loom_paged_plan(const int32_t* table, int64_t table_ld, int64_t max_pages, int64_t n_pages, int64_t page_size,
                               const int32_t* lens, const int32_t* new_tokens, int64_t rows, int64_t n_tokens, int64_t QH,
                               int64_t KVH, int32_t* starts, int32_t* rows_of, int32_t* positions, int64_t* slots,
                               int32_t* shared, void* plan, int64_t plan_bytes, void* stream) {
    return loom_paged_plan_checked(table, table_ld, max_pages, n_pages, page_size, lens, new_tokens, rows, n_tokens, QH, KVH, starts,
                                   rows_of, positions, slots, shared, plan, plan_bytes, nullptr, nullptr, stream);
}

extern "C" int loom_paged_plan_checked(const int32_t* table, int64_t table_ld, int64_t max_pages, int64_t n_pages,
                                       int64_t page_size, const int32_t* lens, const int32_t* new_tokens, int64_t rows,
                                       int64_t n_tokens, int64_t QH, int64_t KVH, int32_t* starts, int32_t* rows_of,
                                       int32_t* positions, int64_t* slots, int32_t* shared, void* plan, int64_t plan_bytes,
                                       int32_t* limit, int32_t* left_out, void* stream) {
    clear_error();
    const char* who = "paged_plan";
    if (int rc = batch_sizes(who, rows, n_tokens, QH, KVH, n_pages, page_size, max_pages, table_ld)) return rc;
    LOOM_CHECK(((table && lens && new_tokens && shared) || rows == 0) && starts && ((rows_of && positions && slots) || n_tokens == 0),
               "%s: a required pointer is NULL", who);
    const int64_t need = loom_paged_plan_bytes(rows, n_tokens, QH, KVH);
    LOOM_CHECK(plan != nullptr && plan_bytes >= need && ((uintptr_t)plan % 64) == 0,
               "%s: a 64-byte aligned plan of %lld bytes is needed, got %lld", who, (long long)need, (long long)plan_bytes);
    PlanArgs a{};
    a.table = table;
    a.table_ld = table_ld;
    a.lens = lens;
    a.fresh = new_tokens;
    a.starts = starts;
    a.rows_of = rows_of;
    a.positions = positions;
    a.shared = shared;
    a.slots_of = slots;
    a.plan = (int32_t*)plan;
    a.limit = limit;
    a.left_out = left_out;
    a.at = pb_layout(rows, n_tokens, QH, KVH);
    a.R = (int)rows;
    a.N = (int)n_tokens;
    a.QH = (int)QH;
    a.KVH = (int)KVH;
    a.G = (int)(QH / KVH);
    a.log_ps = __builtin_ctzll((unsigned long long)page_size);
    a.cap = (int)(max_pages * page_size);
    a.n_pages = (int)n_pages;
    hipStream_t st = (hipStream_t)stream;
    // (about as many segments as threads: see pb_layout)
    const int64_t entries = rows * max_pages, segs = n_tokens * a.G / kPbQ;
    auto blocks = [&](int64_t nt) { return dim3((unsigned)(1 + ceil_div(n_tokens, nt))); };
    if (rows <= 64 && entries <= 1024 && segs <= 64) {
        hipLaunchKernelGGL((paged_plan_kernel<64, true>), blocks(64), dim3(64), 0, st, a);
    } else if (rows <= 256 && entries <= 8192 && segs <= 256) {
        hipLaunchKernelGGL((paged_plan_kernel<256, true>), blocks(256), dim3(256), 0, st, a);
    } else {
        if (rows > 0) hipLaunchKernelGGL(paged_rows_kernel, dim3((unsigned)ceil_div(rows, 16)), dim3(1024), 0, st, a);
        if (int rc = launch_status("loom_paged_plan(rows)")) return rc;
        hipLaunchKernelGGL((paged_plan_kernel<1024, false>), blocks(1024), dim3(1024), 0, st, a);
    }
    return launch_status("loom_paged_plan(plan)");
}

extern "C" int64_t loom_paged_batch_workspace_bytes(int64_t rows, int64_t n_tokens, int64_t QH, int64_t KVH, int64_t HD) {
    if (loom_paged_plan_bytes(rows, n_tokens, QH, KVH) == 0 || HD < 1 || HD > 256) return 0;
    return pb_rec_floats(pb_layout(rows, n_tokens, QH, KVH), KVH, HD) * (int64_t)sizeof(float) + (n_tokens + 15) / 16 * 16;
}

extern "C" int loom_paged_batch_step(int dtype, const void* qkv, int64_t qkv_ld, void* k_pages, void* v_pages,
                                     int64_t page_stride, int64_t token_stride, int64_t head_stride, int64_t n_pages,
                                     int64_t page_size, const int32_t* table, int64_t table_ld, int64_t max_pages,
                                     int64_t rows, const int32_t* rows_of, const int32_t* positions, const int64_t* slots,
                                     const void* plan, int64_t plan_bytes, const float* cos_table, const float* sin_table,
                                     int64_t n_pos, void* q_out, void* c_out, void* kctx_out, int64_t out_ld,
                                     void* workspace, int64_t workspace_bytes, int64_t n_tokens, int64_t QH, int64_t KVH,
                                     int64_t HD, void* stream) {
    clear_error();
    const char* who = "paged_batch_step";
    const BatchCall c{qkv, qkv_ld, k_pages, v_pages, page_stride, token_stride, head_stride, n_pages, page_size, table,
                      table_ld, max_pages, rows, rows_of, positions, slots, plan, plan_bytes, cos_table, sin_table, n_pos,
                      q_out, c_out, kctx_out, out_ld, workspace, workspace_bytes, n_tokens, QH, KVH, HD};
    const int64_t es = dtype == LOOM_F32 ? 4 : 2;
    LOOM_CHECK(dtype == LOOM_F32 || dtype == LOOM_BF16 || dtype == LOOM_F16, "%s: unsupported dtype %d", who, dtype);
    if (int rc = batch_sizes(who, rows, n_tokens, QH, KVH, n_pages, page_size, max_pages, table_ld)) return rc;
    LOOM_CHECK(HD == 8 || HD == 16 || HD == 32 || HD == 64 || HD == 96 || HD == 128 || HD == 256,
               "%s: unsupported head_dim %lld (8, 16, 32, 64, 96, 128 or 256)", who, (long long)HD);
    LOOM_CHECK(token_stride >= HD && token_stride < ((int64_t)1 << 31) / (16 * es) && page_stride >= 0 && head_stride >= 0,
               "%s: bad page strides", who);
    if (n_tokens == 0) return LOOM_OK;
    LOOM_CHECK(qkv && k_pages && v_pages && (table || rows == 0) && rows_of && positions && slots && plan && cos_table &&
                   sin_table && q_out && c_out,
               "%s: a required pointer is NULL", who);
    LOOM_CHECK((token_stride * es) % 16 == 0 && (page_stride * es) % 16 == 0 && (head_stride * es) % 16 == 0 &&
                   (((uintptr_t)k_pages | (uintptr_t)v_pages) % 16) == 0,
               "%s: the pools and their strides must be multiples of 16 bytes", who);
    const int64_t width = (QH + 2 * KVH) * HD;
    LOOM_CHECK(qkv_ld >= width && (qkv_ld * es) % 16 == 0 && ((uintptr_t)qkv % 16) == 0,
               "%s: the rows of qkv must be 16-byte aligned and hold %lld elements (row stride %lld)", who,
               (long long)width, (long long)qkv_ld);
    LOOM_CHECK(out_ld >= QH * HD && (out_ld * es) % 16 == 0, "%s: the output rows are %lld elements apart: %lld at least, and 16-byte aligned",
               who, (long long)out_ld, (long long)(QH * HD));
    LOOM_CHECK((((uintptr_t)q_out | (uintptr_t)c_out | (uintptr_t)kctx_out | (uintptr_t)cos_table | (uintptr_t)sin_table) % 16) == 0,
               "%s: the outputs and the rotary tables must be 16-byte aligned", who);
    LOOM_CHECK(n_pos >= 1, "%s: the rotary tables are empty", who);
    // a launch's threads are counted in 32 bits (blocks of 256)
    LOOM_CHECK((int64_t)pb_layout(rows, n_tokens, QH, KVH).cap_items * KVH < (int64_t)1 << 24,
               "%s: %lld tokens of %lld query heads are too many for one call", who, (long long)n_tokens, (long long)QH);
    const int64_t pn = loom_paged_plan_bytes(rows, n_tokens, QH, KVH);
    LOOM_CHECK(plan_bytes >= pn && ((uintptr_t)plan % 64) == 0, "%s: a 64-byte aligned plan of %lld bytes is needed, got %lld", who,
               (long long)pn, (long long)plan_bytes);
    const int64_t need = loom_paged_batch_workspace_bytes(rows, n_tokens, QH, KVH, HD);
    LOOM_CHECK(workspace != nullptr && workspace_bytes >= need && ((uintptr_t)workspace % 16) == 0,
               "%s: a 16-byte aligned workspace of %lld bytes is needed, got %lld", who, (long long)need,
               (long long)workspace_bytes);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == LOOM_F32) return batch_launch<float>(c, s);
    if (dtype == LOOM_BF16) return batch_launch<bf16_t>(c, s);
    return batch_launch<f16_t>(c, s);
}
