// Attention of one new token per row over a paged key-value cache, for gfx950.
//
// Row b holds n_b tokens, token t in page table[b, t / PS] at place t % PS.
// With s_t = q . k_t / sqrt(HD) over t < n_b:
//   C = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),  Kctx = the same of k_t.
// A row's tokens are split into chunks; each chunk leaves (m, l, C, Kctx) with
// its own maximum m and sum l, and the join weighs them by e^(m - max m).
//
// The rows have lengths of their own that only the device knows, so the host
// launches a fixed number of blocks and every block works out its share from
// lens (make_plan): either chunks of equal size, at most one per block, or, where
// a block has many tiles to do, equal stretches of all rows laid end to end.
#include "attn_tile.h"

namespace loom {

typedef float pg_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 pg_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 pg_f16x8 __attribute__((ext_vector_type(8)));

constexpr int kPgTile = 32;       // tokens of one wave step of the matrix-core form
constexpr int kPgLeast = 1;       // a chunk has 2^kPgLeast tiles at least, one in the vector form
constexpr int kPgStream = 16;     // tiles per block from which the rows are laid end to end
constexpr int kPgRowCost = 6;     // what starting on a row costs a block, in tiles
constexpr int kPgWhole = 512;     // rows of up to so many tokens are not split,
constexpr int kPgWholeVec = 8;    // in the vector form of up to so many steps, if there are few rows
constexpr int kPgMaxRows = 1024;

template <typename T>
struct PagedArgs {
    const T* q;            // STEP: projection rows [q | k | v]; else q [B, QH, HD]
    int64_t q_ld;
    T* kp;
    T* vp;
    int64_t ps_page, ps_tok, ps_head;   // strides in elements
    const int32_t* table;
    int64_t table_ld;
    const int32_t* lens;
    const float* cosv;     // STEP: [n_pos, HD]
    const float* sinv;
    T* q_out;
    T* c_out;
    T* k_out;
    int64_t out_ld;
    float* rec;            // chunk records: [item, QH, 2 HD] then [item, QH, 2]
    int64_t rec_ml;        // float offset of the second part
    int n_pages, log_ps, cap, n_pos;
    int B, QH, KVH, G;
    int slots;             // blocks per kv head to share the work among; 0: a block per row
    int least;             // tiles of a chunk at least: 2^least
    float qscale;
};

// Tokens row b attends to (the new one included when step is 1); 0 for an
// idle row; *bad: the row's position lies past its table or the rotary tables.
__device__ __forceinline__ int row_tokens(const int32_t* lens, int b, int step, int cap, int n_pos,
                                          bool* bad) {
    const int n = lens[b];
    *bad = n >= 0 && (n > cap - step || (step && n >= n_pos));
    return n < 0 || *bad ? 0 : n + step;
}

// Lanes 16 and 32 apart: the two values of each pair in every lane of it
__device__ __forceinline__ float2 pair16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float2 pair32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_16_32(float v) {
    float2 p = pair16(v, v);
    v = fmaxf(p.x, p.y);
    p = pair32(v, v);
    return fmaxf(p.x, p.y);
}
__device__ __forceinline__ float sum_16_32(float v) {
    float2 p = pair16(v, v);
    v = p.x + p.y;
    p = pair32(v, v);
    return p.x + p.y;
}

// The exponents' running reference: it follows the maximum (in powers of two) only
// where that is LAG beyond it, so that the sums are hardly ever rescaled.  A factor of
// 2^8 costs nothing where the weights keep an fp32's range of exponents.
constexpr float kPgLag = 8.0f;
__device__ __forceinline__ float raised(float ref, float most, float lag = kPgLag) { return most > ref + lag ? most : ref; }

// Tiles of a row of n tokens; a row of none counts as one, which writes its outputs.
__device__ __forceinline__ int row_tiles(int n) { return n > 0 ? (n + kPgTile - 1) / kPgTile : 1; }

// How the rows' tiles are shared out.  q > 0: block j takes units j q .. (j+1) q - 1
// of the rows laid end to end, a row being kPgRowCost units and its tiles.  Else a
// row of t tiles is cut into slots * t / total equal chunks (at least one, each of
// 2^least or more), one block each: no more chunks than slots, but for rows
// of less than a chunk (a block more than the device holds at once would run
// after all others).
// End to end no block waits for a longer one, but a block that starts on a row pays
// its rope, its join record and an empty pipeline again (about six tiles: 64 rows of
// 1 to 16384 tokens, 8 kv heads of 128, in us with kPgRowCost 2, 4, 6: 87.9, 85.1,
// 84.1); equal chunks have one start per block.  From how many tiles per block the
// former pays, in us with kPgStream 8, 16, 32: 32 rows of 2176 tokens, 2 kv heads of
// 96, 17.2, 17.6, 17.6; the same in fp32 26.4, 27.2, 26.8; 1 row of 16384, 8 kv heads
// of 128, 21.8, 21.0, 21.0.
// The least chunk, in us with 1, 2, 4 tiles: bf16, 1 row of 2000 tokens, 2 kv heads of
// 96, 11.3, 10.4, 10.5, 4 rows of 900, 8 kv heads of 128, 12.6, 12.5, 12.6 (a wave of
// the block without a tile costs nothing); in the vector form, whose blocks do one
// tile at a time, fp32, 5 rows to 1001, 11.5, 12.3, 14.0.
struct Plan {
    int q, slots, total, least;
};

template <bool STEP>
__device__ __forceinline__ Plan make_plan(const int32_t* lens, int B, int cap, int n_pos, int slots, int least) {
    if (slots == 0) return Plan{0, 0, 1, 0};
    int total = 0;
    bool bad;
    for (int b = threadIdx.x & 63; b < B; b += 64) total += row_tiles(row_tokens(lens, b, STEP, cap, n_pos, &bad));
    total = wave_sum_int(total);
    const bool stream = total >= kPgStream * slots;
    return Plan{stream ? (total + B * kPgRowCost + slots - 1) / slots : 0, slots, total, least};
}

__device__ __forceinline__ int plan_units(const Plan& p, int tiles) {
    if (p.q > 0) return tiles + kPgRowCost;
    const uint32_t n = (uint32_t)tiles * (uint32_t)p.slots / (uint32_t)p.total;      // (< 2^19 * 2^9)
    return max(1, (int)min(n, (uint32_t)(tiles + (1 << p.least) - 1) >> p.least));
}

// A row's place in the plan: the units before it, its tokens
struct PlanRow {
    int row, before, tokens;
    bool bad;
};

// The row that unit x lies in (BY_ROW: row x); row = -1: behind the last.
template <bool STEP, bool BY_ROW>
__device__ __forceinline__ PlanRow plan_find(const Plan& p, const int32_t* lens, int B, int cap, int n_pos, int x) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int b = b0 + lane;
        bool bad = false;
        const int n = b < B ? row_tokens(lens, b, STEP, cap, n_pos, &bad) : 0;
        const int u = b < B ? plan_units(p, row_tiles(n)) : 0;
        const int incl = wave_scan_int(u);
        const int first = base + incl - u;
        const bool mine = b < B && (BY_ROW ? b == x : x >= first && x < first + u);
        const unsigned long long who = __ballot(mine);
        if (who) {
            const int src = __builtin_amdgcn_readfirstlane(__ffsll(who) - 1);
            return PlanRow{b0 + src, __builtin_amdgcn_readlane(first, src), __builtin_amdgcn_readlane(n, src),
                           __builtin_amdgcn_readlane((int)bad, src) != 0};
        }
        base += __builtin_amdgcn_readlane(incl, 63);
    }
    return PlanRow{-1, 0, 0, false};
}

// What block j does of a row: tiles tile0 .. tile1 - 1 (none: tile0 >= tile1),
// as chunk `chunk` of nchunk, whose records start at item0 (block + row along the
// staircase of blocks and rows: a number of its own for each pair).
struct PlanItem {
    int row, tokens, tile0, tile1, chunk, nchunk, item0;
    bool bad;
};

__device__ __forceinline__ PlanItem plan_item(const Plan& p, const PlanRow& r, int j) {
    PlanItem it;
    it.row = r.row;
    it.tokens = r.tokens;
    it.bad = r.bad;
    const int t = row_tiles(r.tokens);
    if (p.q > 0) {
        const int p0 = r.before + kPgRowCost;        // the row's first tile
        const int first = (int)((uint32_t)p0 / (uint32_t)p.q);
        it.nchunk = (int)((uint32_t)(p0 + t - 1) / (uint32_t)p.q) - first + 1;
        it.chunk = j - first;
        it.tile0 = max(j * p.q - p0, 0);
        it.tile1 = min((j + 1) * p.q - p0, t);
        it.item0 = first + r.row;
    } else {
        it.nchunk = plan_units(p, t);
        it.chunk = j - r.before;
        it.tile0 = (int)((uint32_t)it.chunk * (uint32_t)t / (uint32_t)it.nchunk);
        it.tile1 = (int)((uint32_t)(it.chunk + 1) * (uint32_t)t / (uint32_t)it.nchunk);
        it.item0 = r.before;
    }
    return it;
}

// The rows of block j, one after the other: f(PlanItem).
template <bool STEP, typename F>
__device__ __forceinline__ void plan_walk(const int32_t* lens, int B, int cap, int n_pos, int slots, int least, int j,
                                          F f) {
    const Plan p = make_plan<STEP>(lens, B, cap, n_pos, slots, least);
    // end to end, `slots` blocks have all units (and only their j q stays within 32 bits)
    if (p.q > 0 && j >= slots) return;
    PlanRow r = plan_find<STEP, false>(p, lens, B, cap, n_pos, p.q > 0 ? j * p.q : j);
    if (r.row < 0) return;
    while (true) {
        const PlanItem it = plan_item(p, r, j);
        if (it.tile0 < it.tile1) f(it);
        if (p.q == 0) return;
        r.before += plan_units(p, row_tiles(r.tokens));
        if (++r.row >= B || r.before >= (j + 1) * p.q) return;
        r.tokens = __builtin_amdgcn_readfirstlane(row_tokens(lens, r.row, STEP, cap, n_pos, &r.bad));
        r.bad = __builtin_amdgcn_readfirstlane((int)r.bad) != 0;
    }
}

// Element pair helpers by type
template <typename T> struct Mfma16;
template <> struct Mfma16<bf16_t> {
    static constexpr float kLag = kPgLag, kShift = 0.0f;
    __device__ __forceinline__ static pg_f32x4 dot(uint4 a, uint4 b, pg_f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pg_bf16x8, a),
                                                       __builtin_bit_cast(pg_bf16x8, b), c, 0, 0, 0);
    }
    __device__ __forceinline__ static uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
};
template <> struct Mfma16<f16_t> {
    // half's exponents end at 2^15 and its normal values at 2^-14, so the reference lies
    // 2^13 below the maximum it follows and lags by 2^2 at most: weights from 2^-27 of
    // the largest on keep their 11 bits, and what a smaller one loses is at most 2^-38
    // of the largest (2^-14 in a row of 2^24 tokens)
    static constexpr float kLag = 2.0f, kShift = 13.0f;
    __device__ __forceinline__ static pg_f32x4 dot(uint4 a, uint4 b, pg_f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pg_f16x8, a),
                                                      __builtin_bit_cast(pg_f16x8, b), c, 0, 0, 0);
    }
    __device__ __forceinline__ static uint32_t pack(float a, float b) {
        f16_t x, y;
        st(&x, a);
        st(&y, b);
        return (uint32_t)x.x | ((uint32_t)y.x << 16);
    }
};

// x c + y s of the rotation.  For the 16-bit types in 64 bits, where both products are
// exact; rounded to fp32 here and to the type when it is stored, the value is the exact
// one's rounding but where fp32's falls on the middle of two values: of 2^24 random ones
// 1058 of half and 114 of bf16 come out a step beside it (all in fp32 2966 and 477).
template <typename T>
__device__ __forceinline__ float turn(float x, float c, float y, float s) {
    if constexpr (sizeof(T) == 2) return (float)fma((double)x, (double)c, (double)y * (double)s);
    else return fmaf(x, c, y * s);
}

// Eight elements of a head from d0 on (a multiple of 8, as HD / 2 is) as they are
// loaded for the rotation x cos + rotate_half(x) sin: all loads first, so that a
// row's are one wait.
template <typename T>
struct Rope8 {
    uint4 x, y;
    float c[8], s[8];
    bool low;                                        // of the first half: x cos - y sin
    __device__ __forceinline__ void load(const T* head, const float* cr, const float* sr, int d0, int HD) {
        const int half = HD / 2;
        low = d0 < half;
        x = *reinterpret_cast<const uint4*>(head + d0);
        y = *reinterpret_cast<const uint4*>(head + (low ? d0 + half : d0 - half));
        Vec8<float>::load(cr + d0, c);
        Vec8<float>::load(sr + d0, s);
    }
    __device__ __forceinline__ uint4 packed() const {
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float v[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const T xe{(uint16_t)(xs[k] >> (16 * h))}, ye{(uint16_t)(ys[k] >> (16 * h))};
                v[h] = turn<T>(ld(&xe), c[2 * k + h], low ? -ld(&ye) : ld(&ye), s[2 * k + h]);
            }
            o[k] = Mfma16<T>::pack(v[0], v[1]);
        }
        return make_uint4(o[0], o[1], o[2], o[3]);
    }
};

// The end of a chunk: the NW waves' (m, l, C, Kctx) of nh heads from LDS (wave w,
// head j: wm[j][w], wl[j][w], and wacc + ((w * NH + j) * 2 + which) * HD)
// joined into the chunk's record, or into the outputs when it is the row's only
// chunk.  A row of no token gives zeros; NaN weights stay NaN, and a sum of 0 (every
// score is -inf) gives NaN, as the softmax does.
template <int NW, typename T>
__device__ __forceinline__ void paged_finish(const PagedArgs<T>& a, const PlanItem& it, int h0, int nh,
                                             int NH, int HD, bool kctx, bool broken, const float* wm,
                                             const float* wl, const float* wacc) {
    // four sums per thread: of head j, C (which = 0) or Kctx, from d on
    const int quads = HD / 4, per_head = kctx ? 2 * quads : quads;
    for (int k = threadIdx.x; k < nh * per_head; k += blockDim.x) {
        const int j = k / per_head, e = k - j * per_head, which = e >= quads, d = 4 * (e - which * quads), h = h0 + j;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) m = fmaxf(m, wm[j * NW + w]);
        float l = 0.0f;
        pg_f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(wm[j * NW + w] - m);
            const pg_f32x4 x = *reinterpret_cast<const pg_f32x4*>(wacc + (size_t)((w * NH + j) * 2 + which) * HD + d);
            l = fmaf(wl[j * NW + w], f, l);
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = fmaf(x[i], f, c[i]);
        }
        if (broken) l = NAN;
        if (it.nchunk == 1) {
            const float inv = 1.0f / l;
            const bool none = it.tokens <= 0 && !broken;
            T* out = (which ? a.k_out : a.c_out) + (int64_t)it.row * a.out_ld + (int64_t)h * HD + d;
#pragma unroll
            for (int i = 0; i < 4; ++i) st(out + i, none ? 0.0f : c[i] * inv);
        } else {
            const int64_t r = (int64_t)(it.item0 + it.chunk) * a.QH + h;
            *reinterpret_cast<pg_f32x4*>(a.rec + (r * 2 + which) * HD + d) = c;
            if (e == 0) *reinterpret_cast<float2*>(a.rec + a.rec_ml + 2 * r) = make_float2(m, l);
        }
    }
}

// ------------------------------------------------------------------ matrix-core form
// 16-bit types, HD 32 / 64 / 96 / 128, up to 16 query heads per kv head.  NW
// waves, each 32 tokens at a time through LDS tiles of its own (no barrier in the
// loop): S^T = K Q^T, P from the score registers, C = P V and Kctx = P K through
// the transposing LDS read.  A 16-token half of a tile lies in one page (pages
// hold a multiple of 16 tokens), so its base address and its bound are scalar:
// rows past the chunk's end and pages that are missing load zeros.
// Long rows are bound by the reading of K and V, each once for all of a kv head's
// query heads and for both sums: 64 rows of 1 to 16384 tokens, 8 kv heads of 128,
// bf16, 442 MB: 77 us here and 7 in the join, 5.2 TB/s over both (a large copy runs
// at 5.2); half the same; 64 rows of 2048 5.9 TB/s.  Short ones by the chain of first loads: lens,
// table, the row's K; scores; the waves' join: 1 row of 300, 2 kv heads of 96, 7 us of
// which an empty launch is 2.  Two waves per SIMD leave 256 registers, so that the
// next tile's K and V are in flight in registers while the present one is multiplied.
template <typename T, int HD, int NW, bool STEP, bool KCTX>
__global__ void __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
paged_mfma_kernel(PagedArgs<T> a) {
    constexpr int KK = HD / 32, DT = HD / 16, CPR = HD / 8;
    constexpr int NH2 = CPR / 4;              // load instructions per 16-row half
    constexpr int NH = 16;
    struct Tiles {
        gqa_u4 k[kPgTile * CPR];
        gqa_u4 v[kPgTile * CPR];
    };
    constexpr int kTileBytes = NW * (int)sizeof(Tiles);
    constexpr int kRedBytes = NW * NH * (2 + 2 * HD) * (int)sizeof(float);
    __shared__ __align__(16) unsigned char lds[kTileBytes > kRedBytes ? kTileBytes : kRedBytes];
    __shared__ uint4 heads[STEP ? 18 * CPR : 1];      // q of up to 16 heads, k, v of the new token
    using M = Mfma16<T>;
    const int kvh = blockIdx.y, G = a.G;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int lr = lane & 15, lq = lane >> 4;
    const int ps_mask = (1 << a.log_ps) - 1;
    Tiles& tl = reinterpret_cast<Tiles*>(lds)[wave];
    const TileLane<CPR> tln(lq, lr);
    // byte offset of this lane's piece of load i inside a 16-row half
    uint32_t loff[NH2];
#pragma unroll
    for (int i = 0; i < NH2; ++i) {
        const int j = i * 64 + lane, row = j / CPR, c = j - row * CPR;
        loff[i] = (uint32_t)(row * a.ps_tok * (int)sizeof(T)) + 16 * c;
    }
    plan_walk<STEP>(a.lens, a.B, a.cap, a.n_pos, a.slots, a.least, blockIdx.x, [&](const PlanItem& it) {
        const int64_t b = it.row;
        const int pos = it.tokens - 1;
        const int t1 = min(it.tile1 * kPgTile, it.tokens);
        const int ts0 = (it.tile0 + wave) * kPgTile;
        const int32_t* trow = a.table + b * a.table_ld;
        bool broken = it.bad;
        // page of each half of the tile at ts (past the chunk's end: of no use)
        auto pages_of = [&](int ts, int (&pg)[2]) {
#pragma unroll
            for (int h = 0; h < 2; ++h) pg[h] = trow[min(ts + 16 * h, a.cap - 1) >> a.log_ps];
        };
        int pg[2];
        pages_of(ts0, pg);

        // the new token's heads, roped and rounded by one thread per eight elements
        // (q of the block's heads, then k, then v); all waves take q from LDS, and in
        // the block of the row's last chunk the tile that holds the new token takes
        // (k, v) from there: nothing in this launch depends on the row in the pool
        const T* qrow = a.q + b * a.q_ld;
        const bool holds_new = STEP && it.tokens > 0 && it.chunk == it.nchunk - 1;
        constexpr int kNew = 18 * CPR / (NW * 64) + 1;       // rounds for 16 + 2 heads
        Rope8<T> rq[STEP ? kNew : 1];
        int pgn = -1;
        if constexpr (STEP) {
            if (holds_new) pgn = trow[pos >> a.log_ps];
            if (it.tokens > 0) {
                const float* cr = a.cosv + (int64_t)pos * HD;
                const float* sr = a.sinv + (int64_t)pos * HD;
#pragma unroll
                for (int n = 0; n < kNew; ++n) {
                    const int i = tid + n * NW * 64, hh = i / CPR;
                    if (hh >= G + 2) continue;
                    const int h = hh < G ? kvh * G + hh : a.QH + kvh + (hh - G) * a.KVH;
                    rq[n].load(qrow + h * HD, cr, sr, 8 * (i - hh * CPR), HD);
                }
            }
        }
        gqa_u4 kr[2 * NH2], vr[2 * NH2];
        auto load_kv = [&](int ts) {                 // the tile at ts, whose pages are in pg
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int t = ts + 16 * h;
                const int rows = min(16, t1 - t);    // tokens of this half (<= 0: none)
                const int page = __builtin_amdgcn_readfirstlane(pg[h]);
                int bytes = 0;
                int64_t off = 0;
                if (rows > 0) {
                    if ((unsigned)page < (unsigned)a.n_pages) {
                        bytes = ((rows - 1) * (int)a.ps_tok + HD) * (int)sizeof(T);
                        off = (int64_t)page * a.ps_page + (int64_t)(t & ps_mask) * a.ps_tok + kvh * a.ps_head;
                    } else {
                        broken = true;
                    }
                }
                const auto rk_ = __builtin_amdgcn_make_buffer_rsrc((void*)(a.kp + off), (short)0, bytes, kBufferDword3);
                const auto rv_ = __builtin_amdgcn_make_buffer_rsrc((void*)(a.vp + off), (short)0, bytes, kBufferDword3);
#pragma unroll
                for (int i = 0; i < NH2; ++i) {
                    kr[h * NH2 + i] = __builtin_amdgcn_raw_buffer_load_b128(rk_, loff[i], 0, 2);
                    vr[h * NH2 + i] = __builtin_amdgcn_raw_buffer_load_b128(rv_, loff[i], 0, 2);
                }
            }
        };
        load_kv(ts0);
        pages_of(ts0 + NW * kPgTile, pg);

        uint4 qf[KK];                                        // B operand of S^T: head lr, dims 32 kk + 8 lq ..
        if constexpr (STEP) {
            const int page = __builtin_amdgcn_readfirstlane(pgn);
            const bool have = (unsigned)page < (unsigned)a.n_pages;
#pragma unroll
            for (int n = 0; n < kNew; ++n) {
                const int i = tid + n * NW * 64, hh = i / CPR, c = i - hh * CPR;
                if (hh >= G + 2) continue;
                const uint32_t none = M::pack(it.bad ? NAN : 0.0f, it.bad ? NAN : 0.0f);
                uint4 w = make_uint4(none, none, none, none);
                if (it.tokens > 0) w = hh == G + 1 ? rq[n].x : rq[n].packed();
                heads[i] = w;
                if (hh < G) {
                    if (a.q_out != nullptr && it.chunk == 0)
                        *reinterpret_cast<uint4*>(a.q_out + (b * a.QH + kvh * G + hh) * HD + 8 * c) = w;
                } else if (holds_new && have) {
                    const int64_t off = (int64_t)page * a.ps_page + (int64_t)(pos & ps_mask) * a.ps_tok +
                                        kvh * a.ps_head + 8 * c;
                    *reinterpret_cast<uint4*>((hh == G ? a.kp : a.vp) + off) = w;
                }
            }
            lds_barrier();
        }
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            qf[kk] = make_uint4(0, 0, 0, 0);
            if (lr < G)
                qf[kk] = STEP ? heads[lr * CPR + 4 * kk + lq]
                              : *reinterpret_cast<const uint4*>(qrow + (kvh * G + lr) * HD + 32 * kk + 8 * lq);
        }
        const gqa_u4* kn_lds = reinterpret_cast<const gqa_u4*>(heads + G * CPR);
        const gqa_u4* vn_lds = kn_lds + CPR;
        float mh = -INFINITY, lh = 0.0f;
        pg_f32x4 accC[DT], accK[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) accC[dt] = accK[dt] = pg_f32x4{0.f, 0.f, 0.f, 0.f};

        for (int ts = ts0; ts < t1; ts += NW * kPgTile) {
            wave_lds_fence();
            if (holds_new && pos >= ts && pos < ts + kPgTile) {
#pragma unroll
                for (int i = 0; i < 2 * NH2; ++i) {
                    const int j = i * 64 + lane, row = j / CPR, c = j - row * CPR;
                    if (ts + row == pos) {
                        kr[i] = kn_lds[c];
                        vr[i] = vn_lds[c];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2 * NH2; ++i) {
                const int j = i * 64 + lane, row = j / CPR, c = j - row * CPR;
                const int slot = row * CPR + (c ^ kv_swz(row));
                tl.k[slot] = kr[i];
                tl.v[slot] = vr[i];
            }
            const int tn = ts + NW * kPgTile;
            if (tn < t1) {
                load_kv(tn);
                pages_of(tn + NW * kPgTile, pg);
            }
            wave_lds_fence();
            // S^T[token 16 hf + 4 lq + r][head lr]
            pg_f32x4 sc[2];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                sc[hf] = pg_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < KK; ++kk)
                    sc[hf] = M::dot(__builtin_bit_cast(uint4, tile_s_frag<CPR>(tl.k, tln, hf, kk)), qf[kk], sc[hf]);
            }
            float mx = -INFINITY, sv[2][4];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool ok = ts + 16 * hf + 4 * lq + r < t1;
                    sv[hf][r] = ok ? sc[hf][r] * a.qscale : -INFINITY;
                    mx = fmaxf(mx, sv[hf][r]);
                }
            mx = max_16_32(mx);
            const float mnew = raised(mh, mx - M::kShift, M::kLag);
            const float corr = mnew == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mh - mnew);
            float ls = 0.0f, pv[2][4];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    pv[hf][r] = sv[hf][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sv[hf][r] - mnew);
                    ls += pv[hf][r];
                }
            ls = sum_16_32(ls);
            lh = fmaf(lh, corr, ls);
            const bool rescale = corr != 1.0f && mh != -INFINITY;      // (before, the sums are zero)
            mh = mnew;
            // the weights enter the products rounded to the storage type (half a step of
            // it, relative, per weight, down to Mfma16's smallest: below the rounding of
            // the outputs); their sum l is that of the unrounded ones
            const uint4 pa = make_uint4(M::pack(pv[0][0], pv[0][1]), M::pack(pv[0][2], pv[0][3]),
                                        M::pack(pv[1][0], pv[1][1]), M::pack(pv[1][2], pv[1][3]));
            if (__any(rescale)) {
                float cf[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) cf[r] = __shfl(corr, 4 * lq + r, 64);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        accC[dt][r] *= cf[r];
                        if constexpr (KCTX) accK[dt][r] *= cf[r];
                    }
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                accC[dt] = M::dot(pa, tile_tr_frag<CPR>(tl.v, tln, dt), accC[dt]);
                if constexpr (KCTX) accK[dt] = M::dot(pa, tile_tr_frag<CPR>(tl.k, tln, dt), accK[dt]);
            }
        }
        broken = __syncthreads_or(broken);           // and every wave is done with its tiles
        float* wm = reinterpret_cast<float*>(lds);
        float* wl = wm + NW * NH;
        float* wacc = wl + NW * NH;
        if (lq == 0) {
            wm[lr * NW + wave] = mh;
            wl[lr * NW + wave] = lh;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float* acc = wacc + ((wave * NH + 4 * lq + r) * 2) * HD + 16 * dt + lr;
                if (4 * lq + r < G) {
                    acc[0] = accC[dt][r];
                    if constexpr (KCTX) acc[HD] = accK[dt][r];
                }
            }
        __syncthreads();
        paged_finish<NW>(a, it, kvh * G, G, NH, HD, KCTX, broken, wm, wl, wacc);
        __syncthreads();                             // before the next row's tiles
    });
}

// ------------------------------------------------------------------ vector form
// fp32 (whose products stay in fp32) and the head sizes the matrix-core form
// does not take.  LPR lanes per token, each NV groups of four elements (group
// j + LPR v of the row), GT heads per block; scores by a lane-group sum.  The next
// tokens' rows are in flight while the present ones are folded in.  fp32, 32 rows of
// 2176 tokens, 2 kv heads of 96, 107 MB: 27 us with the join, 4.0 TB/s; bound by its
// arithmetic, 2 G products per K and G per V element with no matrix instruction (a
// step of 32 tokens takes 0.8 us).  bf16 heads of 256, 4 kv heads, 285 MB, 54 us, as a
// large copy; 24 query heads on one kv head of 64, 18 MB, 66 us, far from that: six
// blocks of four heads read the rows again and multiply them in fp32.  5 rows of 1 to 1001: 12 us with the join, of which
// about 8 are the first loads, the rope and the waves' join.
template <typename T>
__device__ __forceinline__ void load4(const T* p, float v[4]) {
    if constexpr (sizeof(T) == 4) {
        const pg_f32x4 w = __builtin_nontemporal_load(reinterpret_cast<const pg_f32x4*>(p));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = w[e];
    } else {
        typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));
        const u32x2v w = __builtin_nontemporal_load(reinterpret_cast<const u32x2v*>(p));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const T lo{(uint16_t)(w[e] & 0xffffu)}, hi{(uint16_t)(w[e] >> 16)};
            v[2 * e] = ld(&lo);
            v[2 * e + 1] = ld(&hi);
        }
    }
}

template <typename T, int LPR, int NV, int GT, bool STEP>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
paged_vec_kernel(PagedArgs<T> a) {
    constexpr int HD = LPR * NV * 4, E = NV * 4, NW = 4;
    constexpr int RPW = 64 / LPR, RPB = NW * RPW;       // tokens of a wave / block step
    __shared__ __align__(16) float wm[NW * GT], wl[NW * GT], wacc[NW * GT * 2 * HD];
    __shared__ __align__(16) float heads[(GT + 2) * HD];   // the new token's q, k, v
    const int htiles = (a.G + GT - 1) / GT;
    const int kvh = blockIdx.y / htiles, g0 = (blockIdx.y % htiles) * GT;
    const int nh = min(GT, a.G - g0), h0 = kvh * a.G + g0;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int j = lane % LPR, grp = wave * RPW + lane / LPR;
    const int ps_mask = (1 << a.log_ps) - 1;
    const bool kctx = a.k_out != nullptr;
    plan_walk<STEP>(a.lens, a.B, a.cap, a.n_pos, a.slots, a.least, blockIdx.x, [&](const PlanItem& it) {
        const int64_t b = it.row;
        const int pos = it.tokens - 1;
        const int t0 = it.tile0 * kPgTile, t1 = min(it.tile1 * kPgTile, it.tokens);
        const int32_t* trow = a.table + b * a.table_ld;
        bool broken = it.bad;
        // cached tokens; the new one is folded in from the projection row, first
        const int tc = STEP ? min(t1, pos) : t1;
        auto page_at = [&](int t) { return trow[min(t, a.cap - 1) >> a.log_ps]; };
        const T* qrow = a.q + b * a.q_ld;
        const float* cr = a.cosv + (int64_t)pos * HD;   // read only where tokens > 0
        const float* sr = a.sinv + (int64_t)pos * HD;
        int pg = page_at(t0 + grp);
        // the new token's heads (q of the block's heads, then k, then v) by one thread
        // per four elements; every lane takes what it needs from LDS
        const bool holds_new = STEP && it.tokens > 0 && it.chunk == it.nchunk - 1;
        constexpr int kG4 = HD / 4, kNew = (GT + 2) * kG4 / 256 + 1;
        float xr[kNew][4], yr[kNew][4], cs[kNew][4], sn[kNew][4];
        int pgn = -1;
        if (holds_new) pgn = page_at(pos);
#pragma unroll
        for (int n = 0; n < kNew; ++n) {
            const int i = tid + n * 256, hh = i / kG4, d = 4 * (i - hh * kG4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                xr[n][e] = it.bad ? NAN : 0.0f;
                yr[n][e] = cs[n][e] = sn[n][e] = 0.0f;
            }
            if (hh >= GT + (STEP ? 2 : 0) || (hh < GT && hh >= nh) || (STEP && it.tokens <= 0)) continue;
            const T* head = qrow + (int64_t)(hh < GT ? h0 + hh : a.QH + kvh + (hh - GT) * a.KVH) * HD;
            load4(head + d, xr[n]);
            if constexpr (STEP) {
                load4(head + (d < HD / 2 ? d + HD / 2 : d - HD / 2), yr[n]);
                load4(cr + d, cs[n]);
                load4(sr + d, sn[n]);
            }
        }
        float kv[E], vv[E], kn[E], vn[E];
        // the row of token t, whose page is `page`; false where there is none: the
        // lanes then hold some row of the pool, set to zeros before it is used
        auto load_row = [&](int t, int page, float (&k)[E], float (&v_)[E]) __attribute__((always_inline)) {
            const bool in = t < tc, have = in && (unsigned)page < (unsigned)a.n_pages;
            broken |= in && !have;
            const int64_t off = (have ? (int64_t)page * a.ps_page + (int64_t)(t & ps_mask) * a.ps_tok : 0) + kvh * a.ps_head;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                load4(a.kp + off + 4 * (j + LPR * v), &k[4 * v]);
                load4(a.vp + off + 4 * (j + LPR * v), &v_[4 * v]);
            }
            return have;
        };
        bool ok = load_row(t0 + grp, pg, kv, vv);
        pg = page_at(t0 + grp + RPB);
        const bool have_new = (unsigned)pgn < (unsigned)a.n_pages;
#pragma unroll
        for (int n = 0; n < kNew; ++n) {
            const int i = tid + n * 256, hh = i / kG4, d = 4 * (i - hh * kG4);
            if (hh >= GT + 2) continue;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = xr[n][e];
                if (STEP && hh <= GT && it.tokens > 0)
                    v[e] = round_to<T>(turn<T>(xr[n][e], cs[n][e], d < HD / 2 ? -yr[n][e] : yr[n][e], sn[n][e]));
                heads[4 * i + e] = v[e];
            }
            if constexpr (STEP) {
                T* out = nullptr;
                if (hh < nh && a.q_out != nullptr && it.chunk == 0) {
                    out = a.q_out + (b * a.QH + h0 + hh) * HD + d;
                } else if (hh >= GT && holds_new && have_new && g0 == 0) {
                    out = (hh == GT ? a.kp : a.vp) + (int64_t)pgn * a.ps_page + (int64_t)(pos & ps_mask) * a.ps_tok +
                          kvh * a.ps_head + d;
                }
                if (out != nullptr) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) st(out + e, v[e]);
                }
            }
        }
        lds_barrier();
        auto take = [&](int hh, float (&o)[E]) __attribute__((always_inline)) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[4 * v + e] = heads[hh * HD + 4 * (j + LPR * v) + e];
        };
        float q[GT][E];
#pragma unroll
        for (int g = 0; g < GT; ++g) {
            take(g, q[g]);
#pragma unroll
            for (int e = 0; e < E; ++e) q[g][e] *= a.qscale;
        }
        float m[GT], l[GT], ac[GT][E], ak[GT][E];
#pragma unroll
        for (int g = 0; g < GT; ++g) {
            m[g] = -INFINITY;
            l[g] = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) ac[g][e] = ak[g][e] = 0.0f;
        }
        auto fold = [&](const float (&k)[E], const float (&v_)[E], bool in) __attribute__((always_inline)) {
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                float s = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) s = fmaf(q[g][e], k[e], s);
                s = group_sum<LPR>(s);
                s = in ? s : -INFINITY;
                const float mx = raised(m[g], s);
                const float p = s == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s - mx);
                if (__any(mx != m[g] && m[g] != -INFINITY)) {          // (before, the sums are zero)
                    const float corr = mx == m[g] ? 1.0f : __builtin_amdgcn_exp2f(m[g] - mx);
                    l[g] *= corr;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        ac[g][e] *= corr;
                        ak[g][e] *= corr;
                    }
                }
                l[g] += p;
                m[g] = mx;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    ac[g][e] = fmaf(p, v_[e], ac[g][e]);
                    ak[g][e] = fmaf(p, k[e], ak[g][e]);
                }
            }
        };
        if constexpr (STEP) {
            if (holds_new) {
                broken |= !have_new;
                if (wave == 0) {                     // one lane group of the block
                    take(GT, kn);
                    take(GT + 1, vn);
                    fold(kn, vn, grp == 0);
                }
            }
        }
        for (int t = t0 + grp; t - grp < tc; t += RPB) {           // block-uniform trip count
            const bool okn = load_row(t + RPB, pg, kn, vn);
            pg = page_at(t + 2 * RPB);
            if (!__all(ok)) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    kv[e] = ok ? kv[e] : 0.0f;
                    vv[e] = ok ? vv[e] : 0.0f;
                }
            }
            fold(kv, vv, ok);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                kv[e] = kn[e];
                vv[e] = vn[e];
            }
            ok = okn;
        }
        // join the wave's token groups (lanes LPR apart), then the waves through LDS:
        // lanes 32 apart take the sums of C and of Kctx, lanes 16 apart those of the
        // even and the odd elements, lanes of one row of 16 all of them
        const int which = lane >> 5, odd = (lane >> 4) & 1;
#pragma unroll
        for (int g = 0; g < GT; ++g) {
            float mw = m[g];
            if constexpr (LPR <= 2) mw = fmaxf(mw, dpp<0x122>(mw));         // row_ror 2, 4, 8
            if constexpr (LPR <= 4) mw = fmaxf(mw, dpp<0x124>(mw));
            if constexpr (LPR <= 8) mw = fmaxf(mw, dpp<0x128>(mw));
            mw = max_16_32(mw);
            const float f = mw == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[g] - mw);
            float lw = l[g] * f;
            if constexpr (LPR <= 2) lw += dpp<0x122>(lw);
            if constexpr (LPR <= 4) lw += dpp<0x124>(lw);
            if constexpr (LPR <= 8) lw += dpp<0x128>(lw);
            lw = sum_16_32(lw);
            float h[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float2 p = pair32(ac[g][e] * f, ak[g][e] * f);
                h[e] = p.x + p.y;
            }
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float2 p = pair16(h[e], h[e + 1]);
                float v = p.x + p.y;
                if constexpr (LPR <= 8) v += dpp<0x128>(v);
                if constexpr (LPR <= 4) v += dpp<0x124>(v);
                if constexpr (LPR <= 2) v += dpp<0x122>(v);
                if ((lane & 15) < LPR)
                    wacc[((wave * GT + g) * 2 + which) * HD + 4 * (j + LPR * (e / 4)) + e % 4 + odd] = v;
            }
            if (lane == 0) {
                wm[g * NW + wave] = mw;
                wl[g * NW + wave] = lw;
            }
        }
        broken = __syncthreads_or(broken);
        paged_finish<NW>(a, it, h0, nh, GT, HD, kctx, broken, wm, wl, wacc);
        __syncthreads();                             // before the next row's sums
    });
}

// ------------------------------------------------------------------ the join
// One block per (row, q head): wave w takes the row's chunk records w, w + 4, ..,
// a whole record of 2 HD sums per load, kPgJoin of them in flight; the waves meet
// in LDS.  Rows of one chunk are done already.  Bound by the chain plan, records,
// sums: 32 rows of 2176 tokens, 8 heads, 3.9 us with a launch's 2; eight records
// in flight and four sums per load took 0.5 us off one and one.
constexpr int kPgJoin = 8;

template <typename T, int HD, bool STEP>
__global__ void __launch_bounds__(256)
paged_join_kernel(PagedArgs<T> a) {
    constexpr int NV = HD > 128 ? 2 : 1, NL = HD / 2 / NV;     // lanes of four sums
    __shared__ float wm[4], wl[4];
    __shared__ __align__(16) float wacc[4][2 * HD];
    const Plan p = make_plan<STEP>(a.lens, a.B, a.cap, a.n_pos, a.slots, a.least);
    const PlanRow r0 = plan_find<STEP, true>(p, a.lens, a.B, a.cap, a.n_pos, blockIdx.x);
    const PlanItem it = plan_item(p, r0, 0);
    if (it.nchunk == 1) return;
    const int h = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float M = -INFINITY, L = 0.0f;
    pg_f32x4 acc[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) acc[v] = pg_f32x4{0.f, 0.f, 0.f, 0.f};
    for (int c0 = wave; c0 < it.nchunk; c0 += 4 * kPgJoin) {
        float2 ml[kPgJoin];
        pg_f32x4 x[kPgJoin][NV];
#pragma unroll
        for (int u = 0; u < kPgJoin; ++u) {
            const int64_t r = (int64_t)(it.item0 + min(c0 + 4 * u, it.nchunk - 1)) * a.QH + h;
            ml[u] = *reinterpret_cast<const float2*>(a.rec + a.rec_ml + 2 * r);
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (lane < NL) x[u][v] = *reinterpret_cast<const pg_f32x4*>(a.rec + r * 2 * HD + 4 * (lane + NL * v));
        }
        float mx = M;
#pragma unroll
        for (int u = 0; u < kPgJoin; ++u)
            if (c0 + 4 * u < it.nchunk) mx = fmaxf(mx, ml[u].x);
        const float f = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M - mx);
        L *= f;
#pragma unroll
        for (int v = 0; v < NV; ++v) acc[v] *= f;
#pragma unroll
        for (int u = 0; u < kPgJoin; ++u) {
            if (c0 + 4 * u >= it.nchunk) continue;
            const float w = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ml[u].x - mx);
            L = fmaf(ml[u].y, w, L);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[v][e] = fmaf(x[u][v][e], w, acc[v][e]);
        }
        M = mx;
    }
    if (lane == 0) {
        wm[wave] = M;
        wl[wave] = L;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
        if (lane < NL) *reinterpret_cast<pg_f32x4*>(&wacc[wave][4 * (lane + NL * v)]) = acc[v];
    __syncthreads();
    const int n = a.k_out != nullptr ? 2 * HD : HD;
    for (int k = threadIdx.x; k < n; k += 256) {
        const float m = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
        float l = 0.0f, x = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(wm[w] - m);
            l = fmaf(wl[w], f, l);
            x = fmaf(wacc[w][k], f, x);
        }
        T* out = (k < HD ? a.c_out : a.k_out) + (int64_t)it.row * a.out_ld + (int64_t)h * HD + (k < HD ? k : k - HD);
        st(out, x / l);                              // (a row of more than one chunk has tokens)
    }
}

// ------------------------------------------------------------------ host side

// Blocks per kv head that share the work: as many as the device holds at once
// (two per CU; 32 rows of 2176 tokens in us with 1, 1.5, 2, 3, 4 per CU: 21.0, 17.5,
// 17.4, 20.1, 22.5, and 64 rows of 2048, 8 kv heads of 128: 120.0, 103.3, 90.5, 100.1,
// 95.4).  None where no row can be long: a block per row then does it in one launch.
// Both ways in us, whole rows / split and joined, at 120, 250, 370, 500 tokens:
//   bf16, 4 rows, 2 kv heads of 96      6.0 / 10.0, 7.0 / 10.2,  8.0 / 10.3,  8.7 / 10.3
//   bf16, 4 rows, 8 kv heads of 128     6.8 / 9.9, 8.6 / 10.0, 10.3 / 11.5, 12.0 / 11.7
//   bf16, 32 rows, 8 kv heads of 128    7.6 / 14.2, 10.5 / 15.6, 12.8 / 18.6, 15.1 / 20.3
// and at 900, 2 kv heads of 96: 1 row 11.2 / 10.3, 32 rows 14.2 / 12.5.  The vector
// form takes a block's 4 waves times 64 / LPR tokens per step, so its bound is in steps:
//   fp32, 5 rows, 2 kv heads of 96, 100, 180, 250 tokens   9.6 / 11.6, 10.7 / 11.7, 12.2 / 11.6
//   bf16, 4 rows, 4 kv heads of 256, the same             10.2 / 12.6, 13.3 / 13.0, 17.1 / 13.4
// unless the rows fill the device: fp32, 128 rows of 440, 2 kv heads of 96, 19.8 / 25.7.
static int paged_slots(int64_t cap, int64_t HD, int64_t KVH, bool vec, int64_t B) {
    const int64_t step = HD <= 8 ? 128 : HD <= 16 ? 64 : HD <= 96 ? 32 : 16;     // tokens of a vector block's step
    const int64_t few = kPgWholeVec * step < kPgWhole ? kPgWholeVec * step : kPgWhole;
    if (cap <= (vec && 2 * B * KVH < device_cus() ? few : kPgWhole)) return 0;
    const int64_t n = 2 * (int64_t)device_cus() / KVH;
    return n < 1 ? 1 : (int)n;
}

// Whether the matrix cores do not take the case (see paged_mfma_kernel)
static bool paged_vec(int64_t es, int64_t HD, int64_t G) {
    return es != 2 || G > 16 || !(HD == 32 || HD == 64 || HD == 96 || HD == 128);
}

// Blocks per kv head of a launch, and records of it: one for each pair of a block
// and a row that it works on (at most slots + B, and ceil(tiles / 2^least) a row).
static int64_t paged_items(int64_t B, int64_t slots) { return slots == 0 ? B : B + slots; }

// Waves of a block that does a row alone: eight, so that its tiles are in flight at
// once, but four where a row has no more tiles than that or where the blocks fill
// the device (two of four waves fit a CU, one of eight).  In us, eight / four: 4 rows,
// 2 kv heads of 96, 120 tokens 6.6 / 6.0; 1 row of 450 8.5 / 9.6; 8 kv heads of 128,
// 4 rows of 440 10.4 / 11.8, 32 of 500 16.0 / 15.2, 64 of 440 28.2 / 23.8.
static bool paged_eight(int64_t cap, int64_t blocks) { return cap > 4 * kPgTile && blocks < device_cus(); }

template <typename T, bool STEP>
static int paged_launch(PagedArgs<T>& a, int64_t HD, hipStream_t st) {
    const int64_t items = paged_items(a.B, a.slots);
    a.rec_ml = items * a.QH * 2 * HD;
    const char* who = STEP ? "loom_paged_decode_step" : "loom_paged_decode_attention";
    bool done = false;
    if constexpr (sizeof(T) == 2) {
        const dim3 grid((unsigned)items, (unsigned)a.KVH);
        const bool eight = a.slots == 0 && paged_eight(a.cap, (int64_t)a.B * a.KVH);
#define LOOM_PG_MF1(HDV, NW, KC)                                                                    \
        hipLaunchKernelGGL((paged_mfma_kernel<T, HDV, NW, STEP, KC>), grid, dim3(NW * 64), 0, st, a)
#define LOOM_PG_MF(HDV)                                                                             \
        if (HD == HDV && !paged_vec(sizeof(T), HD, a.G)) {                                          \
            if (eight && a.k_out != nullptr) LOOM_PG_MF1(HDV, 8, true);                             \
            else if (eight) LOOM_PG_MF1(HDV, 8, false);                                             \
            else if (a.k_out != nullptr) LOOM_PG_MF1(HDV, 4, true);                                 \
            else LOOM_PG_MF1(HDV, 4, false);                                                        \
            done = true;                                                                            \
        }
        LOOM_PG_MF(96) LOOM_PG_MF(128) LOOM_PG_MF(64) LOOM_PG_MF(32)
#undef LOOM_PG_MF
#undef LOOM_PG_MF1
    }
#define LOOM_PG_V(LPR, NV, GT)                                                                      \
    if (!done && HD == LPR * NV * 4) {                                                              \
        if (a.G == 1)                                                                               \
            hipLaunchKernelGGL((paged_vec_kernel<T, LPR, NV, 1, STEP>), dim3((unsigned)items, (unsigned)a.KVH), \
                               dim3(256), 0, st, a);                                                \
        else                                                                                        \
            hipLaunchKernelGGL((paged_vec_kernel<T, LPR, NV, GT, STEP>),                            \
                               dim3((unsigned)items, (unsigned)(a.KVH * ((a.G + GT - 1) / GT))), dim3(256), 0, st, a); \
        done = true;                                                                                \
    }
    LOOM_PG_V(8, 3, 4) LOOM_PG_V(16, 2, 4) LOOM_PG_V(8, 2, 4) LOOM_PG_V(8, 1, 4) LOOM_PG_V(4, 1, 4)
    LOOM_PG_V(2, 1, 4) LOOM_PG_V(16, 4, 2)
#undef LOOM_PG_V
    LOOM_CHECK(done, "%s: unsupported head_dim %lld (8, 16, 32, 64, 96, 128 or 256)", who, (long long)HD);
    const int rc = launch_status(who);
    if (rc != LOOM_OK || a.slots == 0) return rc;      // one chunk per row: no join
#define LOOM_PG_J(HDV)                                                                              \
    if (HD == HDV)                                                                                  \
        hipLaunchKernelGGL((paged_join_kernel<T, HDV, STEP>), dim3((unsigned)a.B, (unsigned)a.QH), dim3(256), 0, st, a);
    LOOM_PG_J(96) LOOM_PG_J(128) LOOM_PG_J(64) LOOM_PG_J(32) LOOM_PG_J(16) LOOM_PG_J(8) LOOM_PG_J(256)
#undef LOOM_PG_J
    return launch_status(who);
}

struct PagedCall {
    const void* q;
    int64_t q_ld;
    void *kp, *vp;
    int64_t page_stride, token_stride, head_stride, n_pages, page_size;
    const int32_t* table;
    int64_t table_ld, max_pages;
    const int32_t* lens;
    const float *cosv, *sinv;
    int64_t n_pos;
    void *q_out, *c_out, *k_out;
    int64_t out_ld;
    float* ws;
    int64_t ws_bytes, B, QH, KVH, HD;
};

template <typename T, bool STEP>
static int paged_typed(const PagedCall& c, hipStream_t st) {
    PagedArgs<T> a{};
    a.q = (const T*)c.q;
    a.q_ld = c.q_ld;
    a.kp = (T*)c.kp;
    a.vp = (T*)c.vp;
    a.ps_page = c.page_stride;
    a.ps_tok = c.token_stride;
    a.ps_head = c.head_stride;
    a.table = c.table;
    a.table_ld = c.table_ld;
    a.lens = c.lens;
    a.cosv = c.cosv;
    a.sinv = c.sinv;
    a.q_out = (T*)c.q_out;
    a.c_out = (T*)c.c_out;
    a.k_out = (T*)c.k_out;
    a.out_ld = c.out_ld;
    a.rec = c.ws;
    a.n_pages = (int)c.n_pages;
    a.log_ps = __builtin_ctzll((unsigned long long)c.page_size);
    a.cap = (int)(c.max_pages * c.page_size);
    a.n_pos = (int)min(c.n_pos, (int64_t)1 << 30);
    a.B = (int)c.B;
    a.QH = (int)c.QH;
    a.KVH = (int)c.KVH;
    a.G = (int)(c.QH / c.KVH);
    const bool vec = paged_vec(sizeof(T), c.HD, a.G);
    a.slots = paged_slots(a.cap, c.HD, c.KVH, vec, c.B);
    a.least = vec ? 0 : kPgLeast;
    a.qscale = kLog2e / sqrtf((float)c.HD);
    return paged_launch<T, STEP>(a, c.HD, st);
}

template <bool STEP>
static int paged_call(const char* who, int dtype, const PagedCall& c, void* stream) {
    clear_error();
    const int64_t es = dtype == LOOM_F32 ? 4 : 2;
    LOOM_CHECK(dtype == LOOM_F32 || dtype == LOOM_BF16 || dtype == LOOM_F16, "%s: unsupported dtype %d", who, dtype);
    LOOM_CHECK(c.B >= 0 && c.B <= kPgMaxRows, "%s: 0 to %d rows, got %lld", who, kPgMaxRows, (long long)c.B);
    LOOM_CHECK(c.KVH >= 1 && c.QH >= c.KVH && c.QH % c.KVH == 0 && c.QH <= 1024, "%s: bad heads QH=%lld KVH=%lld",
               who, (long long)c.QH, (long long)c.KVH);
    LOOM_CHECK(c.HD == 8 || c.HD == 16 || c.HD == 32 || c.HD == 64 || c.HD == 96 || c.HD == 128 || c.HD == 256,
               "%s: unsupported head_dim %lld (8, 16, 32, 64, 96, 128 or 256)", who, (long long)c.HD);
    LOOM_CHECK(c.page_size >= 16 && c.page_size <= 1024 && (c.page_size & (c.page_size - 1)) == 0,
               "%s: page_size must be a power of two from 16 to 1024, got %lld", who, (long long)c.page_size);
    LOOM_CHECK(c.n_pages >= 1 && c.n_pages < ((int64_t)1 << 31), "%s: bad n_pages %lld", who, (long long)c.n_pages);
    LOOM_CHECK(c.max_pages >= 1 && c.max_pages <= ((int64_t)1 << 24) / c.page_size && c.table_ld >= c.max_pages,
               "%s: the table must hold 1 page to 2^24 tokens per row (max_pages=%lld, row stride %lld)", who,
               (long long)c.max_pages, (long long)c.table_ld);
    LOOM_CHECK(c.token_stride >= c.HD && c.token_stride < ((int64_t)1 << 31) / (16 * es) && c.page_stride >= 0 &&
                   c.head_stride >= 0,
               "%s: bad page strides", who);
    LOOM_CHECK((c.token_stride * es) % 16 == 0 && (c.page_stride * es) % 16 == 0 && (c.head_stride * es) % 16 == 0 &&
                   (((uintptr_t)c.kp | (uintptr_t)c.vp) % 16) == 0,
               "%s: the pools and their strides must be multiples of 16 bytes", who);
    const int64_t width = STEP ? (c.QH + 2 * c.KVH) * c.HD : c.QH * c.HD;
    LOOM_CHECK(c.q_ld >= width && (c.q_ld * es) % 16 == 0 && ((uintptr_t)c.q % 16) == 0,
               "%s: the rows of %s must be 16-byte aligned and hold %lld elements (row stride %lld)", who,
               STEP ? "qkv" : "q", (long long)width, (long long)c.q_ld);
    LOOM_CHECK(c.out_ld >= c.QH * c.HD, "%s: the output rows are %lld elements apart, fewer than %lld", who,
               (long long)c.out_ld, (long long)(c.QH * c.HD));
    LOOM_CHECK(c.q && c.kp && c.vp && c.table && c.lens && c.c_out, "%s: a required pointer is NULL", who);
    if (STEP) {
        LOOM_CHECK(c.cosv && c.sinv && c.n_pos >= 1, "%s: the rotary tables are missing or empty", who);
        LOOM_CHECK((((uintptr_t)c.cosv | (uintptr_t)c.sinv | (uintptr_t)c.q_out) % 16) == 0,
                   "%s: the rotary tables and q_out must be 16-byte aligned", who);
    }
    const int64_t need = loom_paged_decode_workspace_bytes(c.B, c.max_pages * c.page_size, c.QH, c.KVH, c.HD);
    LOOM_CHECK(c.ws_bytes >= need && (c.ws != nullptr || need == 0) && ((uintptr_t)c.ws % 16) == 0,
               "%s: a 16-byte aligned workspace of %lld bytes is needed, got %lld", who, (long long)need,
               (long long)c.ws_bytes);
    if (c.B == 0) return LOOM_OK;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == LOOM_F32) return paged_typed<float, STEP>(c, s);
    if (dtype == LOOM_BF16) return paged_typed<bf16_t, STEP>(c, s);
    return paged_typed<f16_t, STEP>(c, s);
}

}  // namespace loom

using namespace loom;

extern "C" int64_t loom_paged_decode_workspace_bytes(int64_t B, int64_t capacity, int64_t QH, int64_t KVH,
                                                     int64_t HD) {
    if (B <= 0 || capacity <= 0 || KVH <= 0) return 0;
    // (whatever the type: as for the form that splits first)
    const int64_t slots = paged_slots(capacity, HD, KVH, true, 0);
    return slots == 0 ? 0 : paged_items(B, slots) * QH * (2 + 2 * HD) * (int64_t)sizeof(float);
}

extern "C" int loom_paged_decode_step(int dtype, const void* qkv, int64_t qkv_ld, void* k_pages, void* v_pages,
                                      int64_t page_stride, int64_t token_stride, int64_t head_stride,
                                      int64_t n_pages, int64_t page_size, const int32_t* table, int64_t table_ld,
                                      int64_t max_pages, const int32_t* lens, const float* cos_table,
                                      const float* sin_table, int64_t n_pos, void* q_out, void* c_out,
                                      void* kctx_out, int64_t out_ld, float* workspace, int64_t workspace_bytes,
                                      int64_t B, int64_t QH, int64_t KVH, int64_t HD, void* stream) {
    const PagedCall c{qkv, qkv_ld, k_pages, v_pages, page_stride, token_stride, head_stride, n_pages, page_size,
                      table, table_ld, max_pages, lens, cos_table, sin_table, n_pos, q_out, c_out, kctx_out,
                      out_ld, workspace, workspace_bytes, B, QH, KVH, HD};
    return paged_call<true>("paged_decode_step", dtype, c, stream);
}

extern "C" int loom_paged_decode_attention(int dtype, const void* q, int64_t q_ld, const void* k_pages,
                                           const void* v_pages, int64_t page_stride, int64_t token_stride,
                                           int64_t head_stride, int64_t n_pages, int64_t page_size,
                                           const int32_t* table, int64_t table_ld, int64_t max_pages,
                                           const int32_t* lens, void* c_out, void* kctx_out, int64_t out_ld,
                                           float* workspace, int64_t workspace_bytes, int64_t B, int64_t QH,
                                           int64_t KVH, int64_t HD, void* stream) {
    const PagedCall c{q, q_ld, (void*)k_pages, (void*)v_pages, page_stride, token_stride, head_stride, n_pages,
                      page_size, table, table_ld, max_pages, lens, nullptr, nullptr, 0, nullptr, c_out, kctx_out,
                      out_ld, workspace, workspace_bytes, B, QH, KVH, HD};
    return paged_call<false>("paged_decode_attention", dtype, c, stream);
}
