// Attention of one new token per row over a paged key-value cache, for gfx950.
//
// Row b holds n_b tokens, token t in page table[b, t / PS] at place t % PS.
// With s_t = q . k_t / sqrt(HD) over t < n_b:
//   C = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),  Kctx = the same of k_t.
// A row's tokens are split into chunks; each chunk leaves (m, l, C, Kctx) with
// its own maximum m and sum l, and the join weighs them by e^(m - max m).
//
// The rows have lengths of their own that only the device knows, so the host
// launches a fixed number of blocks and every block works out its share
// (plan_item): chunks of equal size over all rows, as many as fill the device.
#include "attn_tile.h"

namespace loom {

typedef float pg_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 pg_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 pg_f16x8 __attribute__((ext_vector_type(8)));

constexpr int kPgTile = 32;       // tokens of one wave step of the matrix-core form
constexpr int kPgMinTiles = 4;    // tokens of a chunk: at least one tile per wave
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
    int B, QH, KVH, G, target;
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

// The share of a block: which row and which of its chunks.  Every wave works
// it out by itself (64 rows per lane step), so no barrier is needed.
struct PlanItem {
    int row, chunk, nchunk, item0, tokens;   // item0: the record of the row's chunk 0
    bool bad;
};

__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// Tiles per chunk: the rows' tiles over `target` chunks, at least kPgMinTiles.
__device__ __forceinline__ int plan_chunk_tiles(const int32_t* lens, int B, int step, int cap,
                                                int n_pos, int target) {
    const int lane = threadIdx.x & 63;
    int total = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        bool bad;
        const int b = b0 + lane;
        const int n = b < B ? row_tokens(lens, b, step, cap, n_pos, &bad) : 0;
        total += wave_sum_int((n + kPgTile - 1) / kPgTile);
    }
    return max(kPgMinTiles, (total + target - 1) / target);
}

// by_row: the plan of row `want`; else of item `want` (row = -1: none).
template <bool BY_ROW>
__device__ __forceinline__ PlanItem plan_item(const int32_t* lens, int B, int step, int cap,
                                              int n_pos, int target, int want) {
    const int lane = threadIdx.x & 63;
    const int ct = plan_chunk_tiles(lens, B, step, cap, n_pos, target);
    PlanItem it;
    it.row = -1;
    int base = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int b = b0 + lane;
        bool bad = false;
        const int n = b < B ? row_tokens(lens, b, step, cap, n_pos, &bad) : 0;
        const int nch = b < B ? max(1, ((n + kPgTile - 1) / kPgTile + ct - 1) / ct) : 0;
        int incl = nch;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d, 64);
            if (lane >= d) incl += o;
        }
        const int first = base + incl - nch;
        const bool mine = BY_ROW ? b == want : (b < B && want >= first && want < first + nch);
        const unsigned long long who = __ballot(mine);
        if (who) {
            const int src = __ffsll(who) - 1;
            it.row = b0 + src;
            it.nchunk = __builtin_amdgcn_readlane(nch, src);
            it.item0 = __builtin_amdgcn_readlane(first, src);
            it.tokens = __builtin_amdgcn_readlane(n, src);
            it.bad = __builtin_amdgcn_readlane((int)bad, src) != 0;
            it.chunk = want - it.item0;
            return it;
        }
        base += __builtin_amdgcn_readlane(incl, 63);
    }
    return it;
}

// Element pair helpers by type
template <typename T> struct Mfma16;
template <> struct Mfma16<bf16_t> {
    __device__ __forceinline__ static pg_f32x4 dot(uint4 a, uint4 b, pg_f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pg_bf16x8, a),
                                                       __builtin_bit_cast(pg_bf16x8, b), c, 0, 0, 0);
    }
    __device__ __forceinline__ static uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
};
template <> struct Mfma16<f16_t> {
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

// One element d of a head, roped: x cos + rotate_half(x) sin
template <typename T>
__device__ __forceinline__ float paged_rope(const T* head, const float* cr, const float* sr, int d,
                                            int HD) {
    const int half = HD / 2;
    const float x = ld(head + d), y = ld(head + (d < half ? d + half : d - half));
    return fmaf(x, cr[d], (d < half ? -y : y) * sr[d]);
}

// Eight of them from d0 on (a multiple of 8, as HD / 2 is)
template <typename T>
__device__ __forceinline__ void paged_rope8(const T* head, const float* cr, const float* sr, int d0,
                                            int HD, float out[8]) {
    const int half = HD / 2;
    float x[8], y[8], c[8], s[8];
    Vec8<T>::load(head + d0, x);
    Vec8<T>::load(head + (d0 < half ? d0 + half : d0 - half), y);
    Vec8<float>::load(cr + d0, c);
    Vec8<float>::load(sr + d0, s);
    const float sg = d0 < half ? -1.0f : 1.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = fmaf(x[e], c[e], sg * y[e] * s[e]);
}

// The end of a chunk: the four waves' (m, l, C, Kctx) of `g1 - g0` heads from
// LDS (wave w, head j: wm[w][j], wl[w][j], and wacc + ((w * NH + j) * 2 + which) * HD)
// joined into the chunk's record, or into the outputs when it is the row's only
// chunk.  A sum of 0 (no token) gives zeros; NaN weights stay NaN.
template <typename T>
__device__ __forceinline__ void paged_finish(const PagedArgs<T>& a, const PlanItem& it, int h0, int nh,
                                             int NH, int HD, bool kctx, bool broken, const float* wm,
                                             const float* wl, const float* wacc) {
    for (int k = threadIdx.x; k < nh * HD; k += blockDim.x) {
        const int j = k / HD, d = k - j * HD, h = h0 + j;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) m = fmaxf(m, wm[w * NH + j]);
        float l = 0.0f, c = 0.0f, kx = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(wm[w * NH + j] - m);
            const float* acc = wacc + (size_t)((w * NH + j) * 2) * HD + d;
            l = fmaf(wl[w * NH + j], f, l);
            c = fmaf(acc[0], f, c);
            if (kctx) kx = fmaf(acc[HD], f, kx);
        }
        if (broken) l = NAN;
        if (it.nchunk == 1) {
            const float inv = 1.0f / l;
            const int64_t o = (int64_t)it.row * a.out_ld + (int64_t)h * HD + d;
            st(a.c_out + o, l == 0.0f ? 0.0f : c * inv);
            if (kctx) st(a.k_out + o, l == 0.0f ? 0.0f : kx * inv);
        } else {
            const int64_t r = (int64_t)(it.item0 + it.chunk) * a.QH + h;
            a.rec[r * 2 * HD + d] = c;
            if (kctx) a.rec[r * 2 * HD + HD + d] = kx;
            if (d == 0) {
                a.rec[a.rec_ml + 2 * r] = m;
                a.rec[a.rec_ml + 2 * r + 1] = l;
            }
        }
    }
}

// ------------------------------------------------------------------ matrix-core form
// 16-bit types, HD 32 / 64 / 96 / 128, up to 16 query heads per kv head.  Four
// waves, each 32 tokens at a time through LDS tiles of its own (no barrier in the
// loop): S^T = K Q^T, P from the score registers, C = P V and Kctx = P K through
// the transposing LDS read.  A 16-token half of a tile lies in one page (pages
// hold a multiple of 16 tokens), so its base address and its bound are scalar:
// rows past the chunk's end and pages that are missing load zeros.
template <typename T, int HD, bool STEP, bool KCTX>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
paged_mfma_kernel(PagedArgs<T> a) {
    constexpr int KK = HD / 32, DT = HD / 16, CPR = HD / 8;
    constexpr int NH2 = CPR / 4;              // load instructions per 16-row half
    constexpr int NH = 16;
    struct Tiles {
        gqa_u4 k[kPgTile * CPR];
        gqa_u4 v[kPgTile * CPR];
    };
    constexpr int kTileBytes = 4 * (int)sizeof(Tiles);
    constexpr int kRedBytes = 4 * NH * (2 + 2 * HD) * (int)sizeof(float);
    __shared__ __align__(16) unsigned char lds[kTileBytes > kRedBytes ? kTileBytes : kRedBytes];
    __shared__ uint4 knew[HD / 8], vnew[HD / 8];
    using M = Mfma16<T>;
    const int kvh = blockIdx.y;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int lr = lane & 15, lq = lane >> 4;
    const PlanItem it = plan_item<false>(a.lens, a.B, STEP, a.cap, a.n_pos, a.target, blockIdx.x);
    if (it.row < 0) return;
    const int G = a.G;
    const int64_t b = it.row;
    const int pos = it.tokens - 1;
    const int tiles = (it.tokens + kPgTile - 1) / kPgTile;
    const int tile0 = (int)((int64_t)it.chunk * tiles / it.nchunk);
    const int tile1 = (int)((int64_t)(it.chunk + 1) * tiles / it.nchunk);
    const int t1 = min(tile1 * kPgTile, it.tokens);
    const int nstep = (tile1 - tile0 + 3) / 4;
    const int32_t* trow = a.table + b * a.table_ld;
    const int ps_mask = (1 << a.log_ps) - 1;
    Tiles& tl = reinterpret_cast<Tiles*>(lds)[wave];
    const TileLane<CPR> tln(lq, lr);
    bool broken = it.bad;

    // byte offset of this lane's piece of load i inside a 16-row half
    uint32_t loff[NH2];
#pragma unroll
    for (int i = 0; i < NH2; ++i) {
        const int j = i * 64 + lane, row = j / CPR, c = j - row * CPR;
        loff[i] = (uint32_t)(row * a.ps_tok * (int)sizeof(T)) + 16 * c;
    }
    gqa_u4 kr[2 * NH2], vr[2 * NH2];
    auto load_kv = [&](int ts) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int t = ts + 16 * h;
            const int rows = min(16, t1 - t);             // tokens of this half (<= 0: none)
            int bytes = 0;
            int64_t off = 0;
            if (rows > 0) {
                const int page = __builtin_amdgcn_readfirstlane(trow[t >> a.log_ps]);
                if ((unsigned)page < (unsigned)a.n_pages) {
                    bytes = ((rows - 1) * (int)a.ps_tok + HD) * (int)sizeof(T);
                    off = (int64_t)page * a.ps_page + (int64_t)(t & ps_mask) * a.ps_tok + kvh * a.ps_head;
                } else {
                    broken = true;
                }
            }
            const auto rk = __builtin_amdgcn_make_buffer_rsrc((void*)(a.kp + off), (short)0, bytes, kBufferDword3);
            const auto rv = __builtin_amdgcn_make_buffer_rsrc((void*)(a.vp + off), (short)0, bytes, kBufferDword3);
#pragma unroll
            for (int i = 0; i < NH2; ++i) {
                kr[h * NH2 + i] = __builtin_amdgcn_raw_buffer_load_b128(rk, loff[i], 0, 2);
                vr[h * NH2 + i] = __builtin_amdgcn_raw_buffer_load_b128(rv, loff[i], 0, 2);
            }
        }
    };
    const int ts0 = __builtin_amdgcn_readfirstlane((tile0 + wave) * kPgTile);
    load_kv(ts0);

    const T* qrow = a.q + b * a.q_ld;
    const bool holds_new = STEP && it.tokens > 0 && it.chunk == it.nchunk - 1;
    if constexpr (STEP) {
        // the block of the row's last chunk appends this token's (k roped, v) and
        // keeps it in LDS: its own scores take the row from there
        if (holds_new) {
            const int page = __builtin_amdgcn_readfirstlane(trow[pos >> a.log_ps]);
            const bool have = (unsigned)page < (unsigned)a.n_pages;
            if (tid < HD / 8) {
                const T* kh = qrow + (a.QH + kvh) * HD;
                float x[8];
                paged_rope8(kh, a.cosv + (int64_t)pos * HD, a.sinv + (int64_t)pos * HD, 8 * tid, HD, x);
                const uint4 kw = make_uint4(M::pack(x[0], x[1]), M::pack(x[2], x[3]), M::pack(x[4], x[5]),
                                            M::pack(x[6], x[7]));
                const uint4 vw = *reinterpret_cast<const uint4*>(kh + a.KVH * HD + 8 * tid);
                knew[tid] = kw;
                vnew[tid] = vw;
                if (have) {
                    const int64_t off = (int64_t)page * a.ps_page + (int64_t)(pos & ps_mask) * a.ps_tok +
                                        kvh * a.ps_head + 8 * tid;
                    *reinterpret_cast<uint4*>(a.kp + off) = kw;
                    *reinterpret_cast<uint4*>(a.vp + off) = vw;
                }
            }
            lds_barrier();
        }
    }
    // B operand of S^T: q of head lr, dims 32 kk + 8 lq ..
    uint4 qf[KK];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
        uint4 w = make_uint4(0, 0, 0, 0);
        const int d0 = 32 * kk + 8 * lq;
        if (lr < G) {
            const int h = kvh * G + lr;
            if constexpr (STEP) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = it.bad ? NAN : 0.0f;
                if (it.tokens > 0)
                    paged_rope8(qrow + h * HD, a.cosv + (int64_t)pos * HD, a.sinv + (int64_t)pos * HD, d0, HD, x);
                w = make_uint4(M::pack(x[0], x[1]), M::pack(x[2], x[3]), M::pack(x[4], x[5]), M::pack(x[6], x[7]));
                if (a.q_out != nullptr && it.chunk == 0 && wave == 0)
                    *reinterpret_cast<uint4*>(a.q_out + (b * a.QH + h) * HD + d0) = w;
            } else {
                w = *reinterpret_cast<const uint4*>(qrow + h * HD + d0);
            }
        }
        qf[kk] = w;
    }
    const gqa_u4* kn_lds = reinterpret_cast<const gqa_u4*>(knew);
    const gqa_u4* vn_lds = reinterpret_cast<const gqa_u4*>(vnew);
    float mh = -INFINITY, lh = 0.0f;
    pg_f32x4 accC[DT], accK[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) accC[dt] = accK[dt] = pg_f32x4{0.f, 0.f, 0.f, 0.f};

    for (int s = 0; s < nstep; ++s) {
        const int ts = __builtin_amdgcn_readfirstlane(ts0 + s * 4 * kPgTile);
        if (ts >= t1) break;                 // wave-uniform: no tile left for this wave
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
        if (s + 1 < nstep) load_kv(ts + 4 * kPgTile);
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
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mnew = fmaxf(mh, mx);
        const float corr = mnew == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mh - mnew);
        float ls = 0.0f, pv[2][4];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                pv[hf][r] = sv[hf][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sv[hf][r] - mnew);
                ls += pv[hf][r];
            }
        ls += __shfl_xor(ls, 16, 64);
        ls += __shfl_xor(ls, 32, 64);
        lh = fmaf(lh, corr, ls);
        mh = mnew;
        // the weights enter the products rounded to the storage type (half a step of
        // it, relative, per weight: below the rounding of the outputs)
        const uint4 pa = make_uint4(M::pack(pv[0][0], pv[0][1]), M::pack(pv[0][2], pv[0][3]),
                                    M::pack(pv[1][0], pv[1][1]), M::pack(pv[1][2], pv[1][3]));
        if (__any(corr != 1.0f)) {
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
    broken = __syncthreads_or(broken);       // and every wave is done with its tiles
    float* wm = reinterpret_cast<float*>(lds);
    float* wl = wm + 4 * NH;
    float* wacc = wl + 4 * NH;
    if (lq == 0) {
        wm[wave * NH + lr] = mh;
        wl[wave * NH + lr] = lh;
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
    paged_finish(a, it, kvh * G, G, NH, HD, KCTX, broken, wm, wl, wacc);
}

// ------------------------------------------------------------------ vector form
// fp32 (whose products stay in fp32) and the head sizes the matrix-core form
// does not take.  LPR lanes per token, each NV groups of four elements (group
// j + LPR v of the row), GT heads per block; scores by a lane-group sum.
constexpr int kPvUnroll = 2;

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
__global__ void __launch_bounds__(256)
paged_vec_kernel(PagedArgs<T> a) {
    constexpr int HD = LPR * NV * 4, E = NV * 4;
    constexpr int RPW = 64 / LPR, RPB = 4 * RPW;        // tokens of a wave / block step
    __shared__ float wm[4 * GT], wl[4 * GT], wacc[4 * GT * 2 * HD];
    const int htiles = (a.G + GT - 1) / GT;
    const int kvh = blockIdx.y / htiles, g0 = (blockIdx.y % htiles) * GT;
    const int nh = min(GT, a.G - g0), h0 = kvh * a.G + g0;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int j = lane % LPR, grp = wave * RPW + lane / LPR;
    const PlanItem it = plan_item<false>(a.lens, a.B, STEP, a.cap, a.n_pos, a.target, blockIdx.x);
    if (it.row < 0) return;
    const int64_t b = it.row;
    const int pos = it.tokens - 1;
    const int tiles = (it.tokens + kPgTile - 1) / kPgTile;
    const int t0 = (int)((int64_t)it.chunk * tiles / it.nchunk) * kPgTile;
    const int t1 = min((int)((int64_t)(it.chunk + 1) * tiles / it.nchunk) * kPgTile, it.tokens);
    const int32_t* trow = a.table + b * a.table_ld;
    const int ps_mask = (1 << a.log_ps) - 1;
    const bool kctx = a.k_out != nullptr;
    bool broken = it.bad;
    const T* qrow = a.q + b * a.q_ld;
    const float* cr = a.cosv + (int64_t)pos * HD;       // read only where tokens > 0
    const float* sr = a.sinv + (int64_t)pos * HD;

    float q[GT][E];
#pragma unroll
    for (int g = 0; g < GT; ++g)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 4 * (j + LPR * v) + e;
                float x = it.bad ? NAN : 0.0f;
                if (g < nh) {
                    if constexpr (STEP) {
                        if (it.tokens > 0) x = round_to<T>(paged_rope(qrow + (h0 + g) * HD, cr, sr, d, HD));
                        if (a.q_out != nullptr && it.chunk == 0 && grp == 0)
                            st(a.q_out + (b * a.QH + h0 + g) * HD + d, x);
                    } else {
                        x = ld(qrow + (h0 + g) * HD + d);
                    }
                }
                q[g][4 * v + e] = x * a.qscale;
            }
    float m[GT], l[GT], ac[GT][E], ak[GT][E];
#pragma unroll
    for (int g = 0; g < GT; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) ac[g][e] = ak[g][e] = 0.0f;
    }
    auto fold = [&](const float (&kv)[kPvUnroll][E], const float (&vv)[kPvUnroll][E], const bool (&ok)[kPvUnroll]) {
#pragma unroll
        for (int g = 0; g < GT; ++g) {
            float s[kPvUnroll], mx = m[g];
#pragma unroll
            for (int u = 0; u < kPvUnroll; ++u) {
                float x = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) x = fmaf(q[g][e], kv[u][e], x);
                x = group_sum<LPR>(x);
                s[u] = ok[u] ? x : -INFINITY;
                mx = fmaxf(mx, s[u]);
            }
            const float corr = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[g] - mx);
            l[g] *= corr;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                ac[g][e] *= corr;
                ak[g][e] *= corr;
            }
#pragma unroll
            for (int u = 0; u < kPvUnroll; ++u) {
                const float p = s[u] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s[u] - mx);
                l[g] += p;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    ac[g][e] = fmaf(p, vv[u][e], ac[g][e]);
                    ak[g][e] = fmaf(p, kv[u][e], ak[g][e]);
                }
            }
            m[g] = mx;
        }
    };
    // cached tokens; the new one is folded in from the projection row below
    const int tc = STEP ? min(t1, pos) : t1;
    for (int t = t0 + grp; t < tc; t += RPB * kPvUnroll) {
        float kv[kPvUnroll][E], vv[kPvUnroll][E];
        bool ok[kPvUnroll];
        int64_t off[kPvUnroll];
#pragma unroll
        for (int u = 0; u < kPvUnroll; ++u) {
            const int tu = t + RPB * u;
            const int page = tu < tc ? trow[tu >> a.log_ps] : -1;
            ok[u] = (unsigned)page < (unsigned)a.n_pages;
            broken |= tu < tc && !ok[u];
            off[u] = ok[u] ? (int64_t)page * a.ps_page + (int64_t)(tu & ps_mask) * a.ps_tok + kvh * a.ps_head : 0;
        }
#pragma unroll
        for (int u = 0; u < kPvUnroll; ++u)
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (ok[u]) {
                    load4(a.kp + off[u] + 4 * (j + LPR * v), &kv[u][4 * v]);
                    load4(a.vp + off[u] + 4 * (j + LPR * v), &vv[u][4 * v]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) kv[u][4 * v + e] = vv[u][4 * v + e] = 0.0f;
                }
            }
        fold(kv, vv, ok);
    }
    if constexpr (STEP) {
        if (it.tokens > 0 && it.chunk == it.nchunk - 1) {
            const int page = trow[pos >> a.log_ps];
            const bool have = (unsigned)page < (unsigned)a.n_pages;
            broken |= !have;
            if (grp == 0) {                  // one lane group of the block
                float kv[kPvUnroll][E] = {}, vv[kPvUnroll][E] = {};
                bool ok[kPvUnroll] = {};
                const T* kh = qrow + (a.QH + kvh) * HD;
                const T* vh = kh + a.KVH * HD;
                const int64_t off = have ? (int64_t)page * a.ps_page + (int64_t)(pos & ps_mask) * a.ps_tok +
                                               kvh * a.ps_head : 0;
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int d = 4 * (j + LPR * v) + e;
                        kv[0][4 * v + e] = round_to<T>(paged_rope(kh, cr, sr, d, HD));
                        vv[0][4 * v + e] = ld(vh + d);
                        if (have && g0 == 0) {
                            st(a.kp + off + d, kv[0][4 * v + e]);
                            a.vp[off + d] = vh[d];
                        }
                    }
                ok[0] = true;
                fold(kv, vv, ok);
            }
        }
    }
    // join the wave's token groups (lanes LPR apart), then the waves through LDS
#pragma unroll
    for (int g = 0; g < GT; ++g) {
        float mw = m[g];
#pragma unroll
        for (int d = LPR; d < 64; d <<= 1) mw = fmaxf(mw, __shfl_xor(mw, d, 64));
        const float f = mw == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[g] - mw);
        float lw = l[g] * f;
#pragma unroll
        for (int d = LPR; d < 64; d <<= 1) lw += __shfl_xor(lw, d, 64);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float c = ac[g][e] * f, kx = ak[g][e] * f;
#pragma unroll
            for (int d = LPR; d < 64; d <<= 1) {
                c += __shfl_xor(c, d, 64);
                kx += __shfl_xor(kx, d, 64);
            }
            if (lane < LPR) {
                const int dd = 4 * (j + LPR * (e / 4)) + e % 4;
                wacc[((wave * GT + g) * 2) * HD + dd] = c;
                wacc[((wave * GT + g) * 2 + 1) * HD + dd] = kx;
            }
        }
        if (lane == 0) {
            wm[wave * GT + g] = mw;
            wl[wave * GT + g] = lw;
        }
    }
    broken = __syncthreads_or(broken);
    paged_finish(a, it, h0, nh, GT, HD, kctx, broken, wm, wl, wacc);
}

// ------------------------------------------------------------------ the join
// One block per (row, q head), a thread per element: the row's chunk records,
// up to kPgJoin of them in flight.  Rows of one chunk are done already.
constexpr int kPgJoin = 8;

template <typename T>
__global__ void paged_join_kernel(PagedArgs<T> a, int HD, int step) {
    const PlanItem it = plan_item<true>(a.lens, a.B, step, a.cap, a.n_pos, a.target, blockIdx.x);
    const int d = threadIdx.x, h = blockIdx.y;
    if (it.nchunk == 1 || d >= HD) return;
    const bool kctx = a.k_out != nullptr;
    float M = -INFINITY, L = 0.0f, C = 0.0f, K = 0.0f;
    for (int c0 = 0; c0 < it.nchunk; c0 += kPgJoin) {
        float m[kPgJoin], l[kPgJoin], cv[kPgJoin], kv[kPgJoin], mx = M;
#pragma unroll
        for (int u = 0; u < kPgJoin; ++u) {
            const int64_t r = (int64_t)(it.item0 + min(c0 + u, it.nchunk - 1)) * a.QH + h;
            m[u] = a.rec[a.rec_ml + 2 * r];
            l[u] = a.rec[a.rec_ml + 2 * r + 1];
            cv[u] = a.rec[r * 2 * HD + d];
            kv[u] = kctx ? a.rec[r * 2 * HD + HD + d] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < kPgJoin; ++u)
            if (c0 + u < it.nchunk) mx = fmaxf(mx, m[u]);
        const float f = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M - mx);
        L *= f;
        C *= f;
        K *= f;
#pragma unroll
        for (int u = 0; u < kPgJoin; ++u) {
            if (c0 + u >= it.nchunk) continue;
            const float w = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[u] - mx);
            L = fmaf(l[u], w, L);
            C = fmaf(cv[u], w, C);
            K = fmaf(kv[u], w, K);
        }
        M = mx;
    }
    const float inv = 1.0f / L;
    const int64_t o = (int64_t)it.row * a.out_ld + (int64_t)h * HD + d;
    st(a.c_out + o, L == 0.0f ? 0.0f : C * inv);
    if (kctx) st(a.k_out + o, L == 0.0f ? 0.0f : K * inv);
}

// ------------------------------------------------------------------ host side

// Chunks aimed at for each kv head: two blocks per CU in all.
static int paged_target(int64_t KVH) { return (int)max((int64_t)1, 2 * (int64_t)device_cus() / KVH); }

// Most items (chunks over all rows): sum of max(1, ceil(tiles / ct)).
static int64_t paged_items(int64_t B, int64_t cap, int64_t KVH) {
    const int64_t per_row = max((int64_t)1, ceil_div(ceil_div(cap, kPgTile), kPgMinTiles));
    return min(B * per_row, B + paged_target(KVH));
}

template <typename T, bool STEP>
static int paged_launch(PagedArgs<T>& a, int64_t HD, hipStream_t st) {
    const int64_t items = paged_items(a.B, a.cap, a.KVH);
    a.rec_ml = items * a.QH * 2 * HD;
    const char* who = STEP ? "loom_paged_decode_step" : "loom_paged_decode_attention";
    bool done = false;
    if constexpr (sizeof(T) == 2) {
        const dim3 grid((unsigned)items, (unsigned)a.KVH);
#define LOOM_PG_MF(HDV)                                                                             \
        if (!done && HD == HDV && a.G <= 16) {                                                      \
            if (a.k_out != nullptr)                                                                 \
                hipLaunchKernelGGL((paged_mfma_kernel<T, HDV, STEP, true>), grid, dim3(256), 0, st, a);  \
            else                                                                                    \
                hipLaunchKernelGGL((paged_mfma_kernel<T, HDV, STEP, false>), grid, dim3(256), 0, st, a); \
            done = true;                                                                            \
        }
        LOOM_PG_MF(96) LOOM_PG_MF(128) LOOM_PG_MF(64) LOOM_PG_MF(32)
#undef LOOM_PG_MF
    }
#define LOOM_PG_V(LPR, NV)                                                                          \
    if (!done && HD == LPR * NV * 4) {                                                              \
        if (a.G == 1)                                                                               \
            hipLaunchKernelGGL((paged_vec_kernel<T, LPR, NV, 1, STEP>), dim3((unsigned)items, (unsigned)a.KVH), \
                               dim3(256), 0, st, a);                                                \
        else                                                                                        \
            hipLaunchKernelGGL((paged_vec_kernel<T, LPR, NV, 4, STEP>),                             \
                               dim3((unsigned)items, (unsigned)(a.KVH * ((a.G + 3) / 4))), dim3(256), 0, st, a); \
        done = true;                                                                                \
    }
    LOOM_PG_V(8, 3) LOOM_PG_V(8, 4) LOOM_PG_V(8, 2) LOOM_PG_V(8, 1) LOOM_PG_V(4, 1) LOOM_PG_V(2, 1)
    LOOM_PG_V(16, 4)
#undef LOOM_PG_V
    LOOM_CHECK(done, "%s: unsupported head_dim %lld (8, 16, 32, 64, 96, 128 or 256)", who, (long long)HD);
    const int rc = launch_status(who);
    if (rc != LOOM_OK || items <= a.B) return rc;      // one chunk per row: no join
    hipLaunchKernelGGL((paged_join_kernel<T>), dim3((unsigned)a.B, (unsigned)a.QH),
                       dim3((unsigned)(ceil_div(HD, 64) * 64)), 0, st, a, (int)HD, STEP ? 1 : 0);
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
    a.target = paged_target(c.KVH);
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
    LOOM_CHECK(c.max_pages >= 1 && c.max_pages * c.page_size <= ((int64_t)1 << 24) && c.table_ld >= c.max_pages,
               "%s: the table must hold 1 page to 2^24 tokens per row (max_pages=%lld, row stride %lld)", who,
               (long long)c.max_pages, (long long)c.table_ld);
    LOOM_CHECK(c.token_stride >= c.HD && c.token_stride * 16 * es < ((int64_t)1 << 31) && c.page_stride >= 0 &&
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
    const int64_t items = paged_items(B, capacity, KVH);
    return items <= B ? 0 : items * QH * (2 + 2 * HD) * (int64_t)sizeof(float);
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
