// Beam search's selection over beams and vocabulary, and the reordering of
// per-sequence states by the selected parents, for gfx950.
//
// Candidate (row, v) of a group of W beams has the value
//   scores[row] + x[row, v] - logsumexp(x[row]),
// and a finished row offers one candidate, (row, pad) at scores[row].  The
// n_out largest values of each group come out in order, ties by the lowest (row, v).
//
// Within a row the order of values is the order of logits, so the first launch
// needs no logsumexp to pick: each block reads a slice of a row once, keeps its
// exponential sum, and leaves the slice's K largest logits.  The second launch (a
// block per group) joins the sums and ranks the W * slices * K survivors, in
// fp64: two beams' values may lie closer than fp32 resolves.
#include "loom_common.h"

namespace loom {

constexpr int kBeamMaxOut = 64, kBeamMaxBeams = 32;
constexpr int kBeamVec = 8;                       // elements per load
constexpr int kBeamPieces = 4;                    // loads in flight per thread
constexpr int kBeamTile = 256 * kBeamVec * kBeamPieces;   // logits of a block step
constexpr int kBeamMaxCand = 2048;                // survivors of a group

struct BeamArgs {
    const float* scores;        // [groups * W]
    const uint8_t* finished;    // [groups * W] or NULL
    float* out_scores;          // [groups, K]
    int32_t* out_parent;
    int64_t* out_token;
    uint8_t* out_finished;      // or NULL
    int64_t V, ld;
    int W, K, slices, groups;
    int64_t slice_len;
    int64_t eos, pad;
    // survivors [row, slice, K]: logit and token (-1: none); sums [row, slice]
    float* cand_x;
    int32_t* cand_v;
    float* part_m;
    double* part_s;
};

// Order of a logit and its place: larger logit first, then the lower place.
__device__ __forceinline__ uint64_t beam_key(float x, uint32_t place) {
    const uint32_t u = __float_as_uint(x);
    const uint32_t o = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);   // ascending with x
    return ((uint64_t)o << 32) | (uint32_t)~place;
}
__device__ __forceinline__ float beam_key_x(uint64_t k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}

__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t v, int d) {
    const uint32_t lo = __shfl_xor((uint32_t)v, d, 64), hi = __shfl_xor((uint32_t)(v >> 32), d, 64);
    return ((uint64_t)hi << 32) | lo;
}

// The K largest keys of a slice of one row: key 0 means no candidate (a NaN or
// -inf logit).  Per step of kBeamTile logits: the best of each four threads'
// keys; the K-th best of those 64 is a bound that at least K keys reach (each
// is the best of its own four threads) and that only K of the fours can reach,
// so at most K * 4 * 32 keys pass, with the kept ones of earlier steps.  They
// are ranked by counting the larger ones.
template <typename T>
__global__ void __launch_bounds__(256)
beam_row_kernel(const T* __restrict__ logits, BeamArgs a) {
    extern __shared__ uint64_t found[];               // K * 128 + K
    __shared__ uint64_t quad[64], kept[kBeamMaxOut];
    __shared__ float wmax[4];
    __shared__ double wsum[4];
    __shared__ int nfound;
    const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int K = a.K;
    const int64_t rec = (int64_t)row * a.slices + slice;
    if (a.finished != nullptr && a.finished[row]) return;     // its logits are not read
    const T* x = logits + (int64_t)row * a.ld;
    const int64_t v0 = (int64_t)slice * a.slice_len, v1 = min(v0 + a.slice_len, a.V);
    // vector loads start at the last aligned address at or before v0; pieces that
    // are not wholly inside the slice are read element by element
    const int skew = (int)(((uintptr_t)(x + v0) / sizeof(T)) % kBeamVec);
    float m = -INFINITY;                               // of this thread
    double s = 0.0;
    if (tid < K) kept[tid] = 0;
    for (int64_t base = v0 - skew; base < v1; base += kBeamTile) {
        float e[kBeamPieces][kBeamVec];
#pragma unroll
        for (int p = 0; p < kBeamPieces; ++p) {
            const int64_t v = base + (int64_t)(p * 256 + tid) * kBeamVec;
            if (v >= v0 && v + kBeamVec <= v1) {
                Vec8<T>::load(x + v, e[p]);
            } else {
#pragma unroll
                for (int k = 0; k < kBeamVec; ++k) e[p][k] = v + k >= v0 && v + k < v1 ? ld(x + v + k) : -INFINITY;
            }
        }
        // running sum of exponentials
        float mt = m;
        bool nan = false;
#pragma unroll
        for (int p = 0; p < kBeamPieces; ++p)
#pragma unroll
            for (int k = 0; k < kBeamVec; ++k) {
                mt = fmaxf(mt, e[p][k]);
                nan |= e[p][k] != e[p][k];
            }
        float st = 0.0f;
        if (mt != -INFINITY) {
#pragma unroll
            for (int p = 0; p < kBeamPieces; ++p)
#pragma unroll
                for (int k = 0; k < kBeamVec; ++k) st += __builtin_amdgcn_exp2f((e[p][k] - mt) * kLog2e);
            s = s * (double)__builtin_amdgcn_exp2f((m - mt) * kLog2e) + (double)st;
            m = mt;
        }
        if (nan) s = NAN;
        // this thread's best
        float bx = -INFINITY;
        int64_t bv = -1;
#pragma unroll
        for (int p = 0; p < kBeamPieces; ++p)
#pragma unroll
            for (int k = 0; k < kBeamVec; ++k)
                if (e[p][k] > bx) {
                    bx = e[p][k];
                    bv = base + (int64_t)(p * 256 + tid) * kBeamVec + k;
                }
        uint64_t best = bv < 0 ? 0 : beam_key(bx, (uint32_t)bv);
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
            const uint64_t o = shfl_xor_u64(best, d);
            best = o > best ? o : best;
        }
        if ((tid & 3) == 0) quad[tid >> 2] = best;
        if (tid == 0) nfound = 0;
        __syncthreads();
        // the K-th best of the 64 (0 when fewer hold a candidate)
        const uint64_t mine = quad[lane];
        int larger = 0;
#pragma unroll 8
        for (int i = 0; i < 64; ++i) larger += quad[i] > mine;
        const unsigned long long at = __ballot(mine != 0 && larger == K - 1);
        uint64_t bound = 1;                            // every candidate
        if (at) {
            const int l = __ffsll(at) - 1;
            bound = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), l) << 32) |
                    (uint32_t)__builtin_amdgcn_readlane((int)mine, l);
        }
        const uint64_t low = kept[K - 1];
        bound = low > bound ? low : bound;
#pragma unroll
        for (int p = 0; p < kBeamPieces; ++p)
#pragma unroll
            for (int k = 0; k < kBeamVec; ++k) {
                if (!(e[p][k] > -INFINITY)) continue;
                const uint64_t key = beam_key(e[p][k], (uint32_t)(base + (int64_t)(p * 256 + tid) * kBeamVec + k));
                if (key >= bound) found[atomicAdd(&nfound, 1)] = key;
            }
        if (tid < K && kept[tid] >= bound) found[atomicAdd(&nfound, 1)] = kept[tid];
        __syncthreads();
        const int n = nfound;
        if (tid < K) kept[tid] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += 256) {
            const uint64_t key = found[i];
            int rank = 0;
            for (int q = 0; q < n; ++q) rank += found[q] > key;
            if (rank < K) kept[rank] = key;
        }
        __syncthreads();
    }
    // the slice's sum: threads, then waves
    const float mw = wave_max(m);
    double sw = mw == -INFINITY ? s : s * (double)__builtin_amdgcn_exp2f((m - mw) * kLog2e);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sw += __shfl_xor(sw, d, 64);
    if (lane == 0) {
        wmax[wave] = mw;
        wsum[wave] = sw;
    }
    __syncthreads();
    if (tid == 0) {
        const float mb = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
        double sb = 0.0;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            sb += mb == -INFINITY ? wsum[w] : wsum[w] * (double)__builtin_amdgcn_exp2f((wmax[w] - mb) * kLog2e);
        a.part_m[rec] = mb;
        a.part_s[rec] = sb;
    }
    if (tid < K) {
        const uint64_t key = kept[tid];
        a.cand_x[rec * K + tid] = key ? beam_key_x(key) : 0.0f;
        a.cand_v[rec * K + tid] = key ? (int32_t)(uint32_t)~(uint32_t)key : -1;
    }
}

struct BeamCand {
    double value;
    uint32_t place;             // (row in group) * V + token
    uint32_t pad;
};
// larger value first, then the lower place
__device__ __forceinline__ bool beam_before(double v, uint32_t p, double w, uint32_t q) {
    return v > w || (v == w && p < q);
}

__global__ void __launch_bounds__(256)
beam_group_kernel(BeamArgs a, int cap) {
    extern __shared__ BeamCand list[];                // cap
    __shared__ double lse[kBeamMaxBeams], qv[64];
    __shared__ float sc[kBeamMaxBeams];
    __shared__ uint32_t qp[64];
    __shared__ uint8_t fin[kBeamMaxBeams];
    __shared__ int nfound;
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int W = a.W, K = a.K, S = a.slices;
    constexpr uint32_t kNone = 0xffffffffu;
    if (tid < W) {
        const int row = g * W + tid;
        const bool f = a.finished != nullptr && a.finished[row];
        fin[tid] = f;
        sc[tid] = a.scores[row];
        double l = 0.0;
        if (!f) {
            float mb = -INFINITY;
            for (int i = 0; i < S; ++i) mb = fmaxf(mb, a.part_m[(int64_t)row * S + i]);
            for (int i = 0; i < S; ++i) {
                const float mi = a.part_m[(int64_t)row * S + i];
                l += a.part_s[(int64_t)row * S + i] * (mb == -INFINITY ? 1.0 : exp((double)mi - (double)mb));
            }
            l = (double)mb + log(l);                  // -inf: no logit; NaN: a NaN or +inf among them
        }
        lse[tid] = l;
    }
    if (tid == 0) nfound = 0;
    __syncthreads();
    const int n = W * S * K;
    auto candidate = [&](int i, double* v, uint32_t* p) {
        const int w = i / (S * K), k = i - w * S * K;
        *v = -INFINITY;
        *p = kNone;
        double value;
        uint32_t place;
        if (fin[w]) {
            if (k != 0) return;
            value = (double)sc[w];
            place = (uint32_t)(w * a.V + a.pad);
        } else {
            const int64_t r = (int64_t)(g * W + w) * S * K + k;
            const int32_t tok = a.cand_v[r];
            if (tok < 0) return;
            value = ((double)a.cand_x[r] - lse[w]) + (double)sc[w];
            place = (uint32_t)(w * a.V + tok);
        }
        if (!(value > -INFINITY && value < INFINITY)) return;     // NaN as well
        *v = value;
        *p = place;
    };
    double bv = -INFINITY;
    uint32_t bp = kNone;
    for (int i = tid; i < n; i += 256) {
        double v;
        uint32_t p;
        candidate(i, &v, &p);
        if (p != kNone && (bp == kNone || beam_before(v, p, bv, bp))) {
            bv = v;
            bp = p;
        }
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
        const double ov = __shfl_xor(bv, d, 64);
        const uint32_t op = __shfl_xor(bp, d, 64);
        if (op != kNone && (bp == kNone || beam_before(ov, op, bv, bp))) {
            bv = ov;
            bp = op;
        }
    }
    if ((tid & 3) == 0) {
        qv[tid >> 2] = bv;
        qp[tid >> 2] = bp;
    }
    __syncthreads();
    const double mv = qv[lane];
    const uint32_t mp = qp[lane];
    int larger = 0;
    for (int i = 0; i < 64; ++i) larger += qp[i] != kNone && beam_before(qv[i], qp[i], mv, mp);
    const unsigned long long at = __ballot(mp != kNone && larger == K - 1);
    double tv = -INFINITY;
    uint32_t tp = kNone;
    if (at) {
        const int l = __ffsll(at) - 1;
        tv = __shfl(mv, l, 64);
        tp = __shfl(mp, l, 64);
    }
    for (int i = tid; i < n; i += 256) {
        double v;
        uint32_t p;
        candidate(i, &v, &p);
        if (p == kNone || beam_before(tv, tp, v, p)) continue;     // below the bound
        const int k = atomicAdd(&nfound, 1);
        if (k < cap) list[k] = BeamCand{v, p, 0};
    }
    __syncthreads();
    const int m = min(nfound, cap);
    for (int i = tid; i < m; i += 256) {
        const BeamCand c = list[i];
        int rank = 0;
        for (int q = 0; q < m; ++q) rank += beam_before(list[q].value, list[q].place, c.value, c.place);
        if (rank < K) {
            const int64_t o = (int64_t)g * K + rank;
            const int w = (int)(c.place / (uint32_t)a.V);
            const int64_t tok = c.place - (int64_t)w * a.V;
            a.out_scores[o] = (float)c.value;
            a.out_parent[o] = g * W + w;
            a.out_token[o] = tok;
            if (a.out_finished != nullptr) a.out_finished[o] = fin[w] || tok == a.eos;
        }
    }
    // fewer candidates than places: no parent but the group's first row
    for (int k = m + tid; k < K; k += 256) {
        const int64_t o = (int64_t)g * K + k;
        a.out_scores[o] = -INFINITY;
        a.out_parent[o] = g * W;
        a.out_token[o] = a.pad;
        if (a.out_finished != nullptr) a.out_finished[o] = 0;
    }
}

// ------------------------------------------------------------------ reorder

constexpr int kReorderMax = 16, kReorderRows = 1024;

struct ReorderSeg {
    char* p;
    int64_t row_stride, outer_stride, row_bytes;
    int vec, slices, block0;    // bytes per access; column slices per outer index
};
struct ReorderArgs {
    ReorderSeg seg[kReorderMax];
    const int32_t* parent;
    int nseg, R, tx_log;
};

// Row r of every tensor becomes the former row parent[r].  A block owns a slice
// of columns of one tensor for all rows: every thread reads its rows' new
// values, the block meets, every thread writes, so no second buffer is needed.
// Rows that stay, and rows whose parent is no row, are not touched.
template <typename V, int RPT, int NT>
__device__ __forceinline__ void reorder_slice(const ReorderSeg& s, const int32_t* parent, int R, int tx_log,
                                              int slice, int64_t outer) {
    const int TX = 1 << tx_log, TY = NT >> tx_log;
    const int tx = threadIdx.x & (TX - 1), ty = threadIdx.x >> tx_log;
    const int64_t col = ((int64_t)slice * TX + tx) * sizeof(V);
    char* base = s.p + outer * s.outer_stride + col;
    const bool in = col < s.row_bytes;
    V val[RPT];
    bool move[RPT];
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
        const int r = ty + k * TY;
        const int p = in && r < R ? parent[r] : -1;
        move[k] = p >= 0 && p < R && p != r;
        if (move[k]) val[k] = *reinterpret_cast<const V*>(base + p * s.row_stride);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < RPT; ++k)
        if (move[k]) *reinterpret_cast<V*>(base + (int64_t)(ty + k * TY) * s.row_stride) = val[k];
}

template <int RPT, int NT>
__global__ void __launch_bounds__(NT)
reorder_rows_kernel(ReorderArgs a) {
    int i = 0;
    while (i + 1 < a.nseg && (int)blockIdx.x >= a.seg[i + 1].block0) ++i;
    const ReorderSeg& s = a.seg[i];
    const int k = blockIdx.x - s.block0;
    const int slice = k % s.slices;
    const int64_t outer = k / s.slices;
    if (s.vec == 16) reorder_slice<u32x4, RPT, NT>(s, a.parent, a.R, a.tx_log, slice, outer);
    else if (s.vec == 4) reorder_slice<uint32_t, RPT, NT>(s, a.parent, a.R, a.tx_log, slice, outer);
    else reorder_slice<uint8_t, RPT, NT>(s, a.parent, a.R, a.tx_log, slice, outer);
}

// ------------------------------------------------------------------ host side

// Slices of a row: enough blocks for the device, each at least a quarter of a
// step's logits, and few enough that a group's survivors fit one block.
static int64_t beam_slices(int64_t rows, int64_t W, int64_t V, int64_t K) {
    int64_t s = ceil_div(4 * (int64_t)device_cus(), rows);
    const int64_t most = ceil_div(V, kBeamTile / 4), fit = kBeamMaxCand / (W * K);
    s = s < most ? s : most;
    s = s < fit ? s : fit;
    return s < 1 ? 1 : s;
}

}  // namespace loom

using namespace loom;

extern "C" int64_t loom_beam_select_workspace_bytes(int64_t groups, int64_t beams, int64_t V, int64_t n_out) {
    if (groups <= 0 || beams <= 0 || V <= 0 || n_out <= 0) return 0;
    const int64_t recs = groups * beams * beam_slices(groups * beams, beams, V, n_out);
    return recs * (8 + 4 + 8 * n_out) + 16;
}

extern "C" int loom_beam_select(int dtype, const void* logits, int64_t logits_ld, const float* scores,
                                const uint8_t* finished, float* out_scores, int32_t* out_parent,
                                int64_t* out_token, uint8_t* out_finished, int64_t groups, int64_t beams,
                                int64_t V, int64_t n_out, int64_t eos_id, int64_t pad_id, void* workspace,
                                int64_t workspace_bytes, void* stream) {
    clear_error();
    const char* who = "beam_select";
    LOOM_CHECK(dtype == LOOM_F32 || dtype == LOOM_BF16 || dtype == LOOM_F16, "%s: unsupported dtype %d", who, dtype);
    LOOM_CHECK(groups >= 0 && groups <= 65535 && beams >= 1 && beams <= kBeamMaxBeams && groups * beams <= 65535,
               "%s: 1 to %d beams and at most 65535 rows, got %lld groups of %lld", who, kBeamMaxBeams,
               (long long)groups, (long long)beams);
    LOOM_CHECK(V >= 1 && V <= ((int64_t)1 << 24) && logits_ld >= V, "%s: a vocabulary of 1 to 2^24, got %lld (row stride %lld)",
               who, (long long)V, (long long)logits_ld);
    LOOM_CHECK(n_out >= 1 && n_out <= kBeamMaxOut && n_out <= beams * V,
               "%s: n_out must be 1 to %d and at most beams * V, got %lld", who, kBeamMaxOut, (long long)n_out);
    LOOM_CHECK(pad_id >= 0 && pad_id < V, "%s: pad_id must lie in [0, %lld), got %lld", who, (long long)V, (long long)pad_id);
    LOOM_CHECK(logits && scores && out_scores && out_parent && out_token, "%s: a required pointer is NULL", who);
    const int64_t need = loom_beam_select_workspace_bytes(groups, beams, V, n_out);
    LOOM_CHECK(workspace_bytes >= need && (workspace != nullptr || need == 0) && ((uintptr_t)workspace % 16) == 0,
               "%s: a 16-byte aligned workspace of %lld bytes is needed, got %lld", who, (long long)need,
               (long long)workspace_bytes);
    if (groups == 0) return LOOM_OK;
    BeamArgs a{};
    a.scores = scores;
    a.finished = finished;
    a.out_scores = out_scores;
    a.out_parent = out_parent;
    a.out_token = out_token;
    a.out_finished = out_finished;
    a.V = V;
    a.ld = logits_ld;
    a.W = (int)beams;
    a.K = (int)n_out;
    a.groups = (int)groups;
    const int64_t rows = groups * beams, S = beam_slices(rows, beams, V, n_out), recs = rows * S;
    a.slice_len = ceil_div(ceil_div(V, S), kBeamVec) * kBeamVec;
    a.slices = (int)S;
    a.eos = eos_id;
    a.pad = pad_id;
    a.part_s = (double*)workspace;
    a.part_m = (float*)(a.part_s + recs);
    a.cand_x = a.part_m + recs;
    a.cand_v = (int32_t*)(a.cand_x + recs * n_out);
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)S, (unsigned)rows);
    const unsigned lds = (unsigned)((n_out * 128 + n_out) * sizeof(uint64_t));
    if (dtype == LOOM_F32)
        hipLaunchKernelGGL((beam_row_kernel<float>), grid, dim3(256), lds, st, (const float*)logits, a);
    else if (dtype == LOOM_BF16)
        hipLaunchKernelGGL((beam_row_kernel<bf16_t>), grid, dim3(256), lds, st, (const bf16_t*)logits, a);
    else
        hipLaunchKernelGGL((beam_row_kernel<f16_t>), grid, dim3(256), lds, st, (const f16_t*)logits, a);
    if (int rc = launch_status("loom_beam_select(rows)")) return rc;
    // at most K fours of threads reach the bound, each with its share of the survivors
    const int64_t n = beams * S * n_out, pass = n_out * 4 * ceil_div(n, 256), cap = pass < n ? pass : n;
    hipLaunchKernelGGL(beam_group_kernel, dim3((unsigned)groups), dim3(256), (unsigned)(cap * sizeof(BeamCand)), st, a,
                       (int)cap);
    return launch_status("loom_beam_select(groups)");
}

extern "C" int loom_reorder_rows(int64_t n, void* const* tensors, const int64_t* outer, const int64_t* outer_stride,
                                 const int64_t* row_stride, const int64_t* row_bytes, const int32_t* parent,
                                 int64_t rows, void* stream) {
    clear_error();
    const char* who = "reorder_rows";
    LOOM_CHECK(n >= 0 && n <= kReorderMax, "%s: at most %d tensors, got %lld", who, kReorderMax, (long long)n);
    LOOM_CHECK(rows >= 0 && rows <= kReorderRows, "%s: 0 to %d rows, got %lld", who, kReorderRows, (long long)rows);
    if (n == 0 || rows == 0) return LOOM_OK;
    LOOM_CHECK(tensors && outer && outer_stride && row_stride && row_bytes && parent, "%s: a required pointer is NULL", who);
    ReorderArgs a{};
    a.parent = parent;
    a.R = (int)rows;
    // threads across a slice: as many rows at once as there are, at least 16 across
    int nt = rows > 256 ? 1024 : 256, ty = 1;
    while (ty < rows && ty < nt / 16) ty *= 2;
    const int tx = nt / ty;
    a.tx_log = __builtin_ctz((unsigned)tx);
    int64_t blocks = 0;
    for (int64_t i = 0; i < n; ++i) {
        LOOM_CHECK(outer[i] >= 0 && row_bytes[i] >= 0 && row_stride[i] >= row_bytes[i] && outer_stride[i] >= 0,
                   "%s: bad shape of tensor %lld", who, (long long)i);
        if (outer[i] == 0 || row_bytes[i] == 0) continue;
        LOOM_CHECK(tensors[i] != nullptr, "%s: tensor %lld is NULL", who, (long long)i);
        const uint64_t all = (uint64_t)(uintptr_t)tensors[i] | (uint64_t)row_stride[i] | (uint64_t)row_bytes[i] |
                             (outer[i] > 1 ? (uint64_t)outer_stride[i] : 0);
        ReorderSeg& s = a.seg[a.nseg++];
        s.p = (char*)tensors[i];
        s.row_stride = row_stride[i];
        s.outer_stride = outer_stride[i];
        s.row_bytes = row_bytes[i];
        s.vec = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
        s.slices = (int)ceil_div(row_bytes[i], (int64_t)s.vec * tx);
        s.block0 = (int)blocks;
        blocks += s.slices * outer[i];
        LOOM_CHECK(blocks < ((int64_t)1 << 31) && ceil_div(row_bytes[i], (int64_t)s.vec * tx) < ((int64_t)1 << 31),
                   "%s: too much data for one call", who);
    }
    if (blocks == 0) return LOOM_OK;
    const int rpt = (int)ceil_div(rows, ty);
    const dim3 grid((unsigned)blocks);
    hipStream_t st = (hipStream_t)stream;
    if (nt == 1024) hipLaunchKernelGGL((reorder_rows_kernel<16, 1024>), grid, dim3(1024), 0, st, a);
    else if (rpt <= 1) hipLaunchKernelGGL((reorder_rows_kernel<1, 256>), grid, dim3(256), 0, st, a);
    else if (rpt <= 2) hipLaunchKernelGGL((reorder_rows_kernel<2, 256>), grid, dim3(256), 0, st, a);
    else if (rpt <= 4) hipLaunchKernelGGL((reorder_rows_kernel<4, 256>), grid, dim3(256), 0, st, a);
    else if (rpt <= 8) hipLaunchKernelGGL((reorder_rows_kernel<8, 256>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((reorder_rows_kernel<16, 256>), grid, dim3(256), 0, st, a);
    return launch_status("loom_reorder_rows");
}
