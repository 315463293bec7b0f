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
constexpr int kBeamPieces = 4;                    // loads of a thread per step
constexpr int kBeamTile = 256 * kBeamVec * kBeamPieces;   // logits of a block step
constexpr int kBeamMaxCand = 2048;                // survivors of a group, from all its slices
constexpr int kBeamWhole = 32768;                 // logits of a group that one block of 1024 takes
constexpr int kBeamWholeOut = 32, kBeamWholeBeams = 16;

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

// Order of a logit and its place: larger logit first, then the lower place.  The two
// zeros are one value: their keys differ by the place alone, as the comparisons of
// floats (the bests, the bound) take them.
__device__ __forceinline__ uint64_t beam_key(float x, uint32_t place) {
    const uint32_t u = x == 0.0f ? 0u : __float_as_uint(x);
    const uint32_t o = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);   // ascending with x
    return ((uint64_t)o << 32) | (uint32_t)~place;
}
__device__ __forceinline__ float beam_key_x(uint64_t k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}

// the least logit that reaches a bound (1: every candidate does)
__device__ __forceinline__ float beam_low(uint64_t bound) {
    return bound > 1 ? beam_key_x(bound) : -3.402823466e38f;
}

// Lane permutations of 64-bit values inside rows of 16 lanes (see dpp): each step
// pairs the halves of twice the group, so reductions over 2, 4, 8, 16 lanes are
// the first 1, 2, 3, 4 of them.
template <int CTRL>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
    const int lo = (int)v, hi = (int)(v >> 32);
    return ((uint64_t)(uint32_t)__builtin_amdgcn_update_dpp(hi, hi, CTRL, 0xF, 0xF, false) << 32) |
           (uint32_t)__builtin_amdgcn_update_dpp(lo, lo, CTRL, 0xF, 0xF, false);
}
template <int CTRL>
__device__ __forceinline__ int dpp_i32(int v) {
    return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xF, 0xF, false);
}
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    return __builtin_bit_cast(double, dpp_u64<CTRL>(__builtin_bit_cast(uint64_t, v)));
}
__device__ __forceinline__ uint64_t readlane_u64(uint64_t v, int l) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((int)v, l);
}
__device__ __forceinline__ double readlane_f64(double v, int l) {
    return __builtin_bit_cast(double, readlane_u64(__builtin_bit_cast(uint64_t, v), l));
}
// the largest of each aligned group of g = 1, 2, 4, 8 or 16 lanes
__device__ __forceinline__ uint64_t group_max_u64(uint64_t v, int g) {
    if (g >= 2) v = max(v, dpp_u64<kDppQuad1032>(v));
    if (g >= 4) v = max(v, dpp_u64<kDppQuad2301>(v));
    if (g >= 8) v = max(v, dpp_u64<kDppHalfMirror>(v));
    if (g >= 16) v = max(v, dpp_u64<kDppMirror>(v));
    return v;
}
__device__ __forceinline__ int group_sum_int(int v, int g) {
    if (g >= 2) v += __builtin_amdgcn_update_dpp(0, v, kDppQuad1032, 0xF, 0xF, false);
    if (g >= 4) v += __builtin_amdgcn_update_dpp(0, v, kDppQuad2301, 0xF, 0xF, false);
    if (g >= 8) v += __builtin_amdgcn_update_dpp(0, v, kDppHalfMirror, 0xF, 0xF, false);
    if (g >= 16) v += __builtin_amdgcn_update_dpp(0, v, kDppMirror, 0xF, 0xF, false);
    return v;
}
__device__ __forceinline__ double wave_sum_f64(double v) {
    v += dpp_f64<kDppQuad1032>(v);
    v += dpp_f64<kDppQuad2301>(v);
    v += dpp_f64<kDppHalfMirror>(v);
    v += dpp_f64<kDppMirror>(v);
    return (readlane_f64(v, 0) + readlane_f64(v, 16)) + (readlane_f64(v, 32) + readlane_f64(v, 48));
}

// Eight logits as loaded, from place v on; places from v1 on hold -inf.  Rows start
// at any element: which thread sums what goes by the place alone, so that equal
// rows have equal sums (and their candidates tie) wherever they lie.
template <typename T>
struct BeamPiece {
    static constexpr int NW = (int)sizeof(T) * kBeamVec / 4;
    uint32_t w[NW];
    __device__ __forceinline__ void load_whole(const T* x, int v) {
#pragma unroll
        for (int i = 0; i < NW / 4; ++i) {
            u32x4 q;                                 // one load, of any alignment
            __builtin_memcpy(&q, reinterpret_cast<const char*>(x) + ((uint32_t)v * (uint32_t)sizeof(T) + 16 * i), 16);
#pragma unroll
            for (int k = 0; k < 4; ++k) w[4 * i + k] = q[k];
        }
    }
    __device__ __forceinline__ void load(const T* x, int v, int v1) {
        if (v + kBeamVec <= v1) {
            load_whole(x, v);
            return;
        }
        constexpr uint32_t ninf = std::is_same<T, float>::value    ? 0xff800000u
                                  : std::is_same<T, bf16_t>::value ? 0xff80ff80u
                                                                   : 0xfc00fc00u;
#pragma unroll
        for (int i = 0; i < NW; ++i) w[i] = ninf;
#pragma unroll
        for (int k = 0; k < kBeamVec; ++k) {
            if (v + k >= v1) continue;
            if constexpr (sizeof(T) == 4) {
                w[k] = __float_as_uint(x[v + k]);
            } else {
                const uint32_t h = x[v + k].x;
                w[k / 2] = (k & 1) ? (w[k / 2] & 0xffffu) | (h << 16) : (w[k / 2] & 0xffff0000u) | h;
            }
        }
    }
    __device__ __forceinline__ float get(int k) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[k]);
        } else {
            const T t{(uint16_t)(w[k / 2] >> (16 * (k & 1)))};
            return ld(&t);
        }
    }
};

// The largest of three; a NaN gives way.  (fmaxf would first pass each loaded value
// through an instruction of its own that quiets signalling NaNs; here such a one may
// come out instead, or hide what came before it, in a row whose sum is NaN and that
// has no candidate.  What passes in such a row may be more than the bound promises,
// so the lists take no key behind their end.)
__device__ __forceinline__ float beam_max3(float a, float b, float c) {
    float d;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}

// A thread's logits of one step: place of element k of piece p is v + p * stride + k.
template <typename T>
struct BeamStep {
    BeamPiece<T> e[kBeamPieces];
    float top[kBeamPieces];                            // largest of each piece (NaNs apart)
    __device__ __forceinline__ void maxima() {
#pragma unroll
        for (int p = 0; p < kBeamPieces; ++p) {
            top[p] = beam_max3(e[p].get(0), e[p].get(1), e[p].get(1));
#pragma unroll
            for (int k = 2; k < kBeamVec; k += 2) top[p] = beam_max3(top[p], e[p].get(k), e[p].get(k + 1));
        }
    }
    __device__ __forceinline__ float most() const {
        return beam_max3(beam_max3(top[0], top[1], top[2]), top[3], top[3]);
    }
    // Running maximum and sum of exponentials.  A NaN makes the sum NaN, and so does
    // +inf; the maximum stays -inf while there is no other logit.  A wave passes over
    // pieces that lie behind v1.
    __device__ __forceinline__ void sum(float& m, double& s, int v, int stride, int v1) const {
        const int first = __builtin_amdgcn_readfirstlane(v);
        const float mt = fmaxf(m, most());
        const float at = mt == -INFINITY ? 0.0f : mt;
        float st = 0.0f;
#pragma unroll
        for (int p = 0; p < kBeamPieces; ++p)
            if (first + p * stride < v1)
#pragma unroll
                for (int k = 0; k < kBeamVec; ++k) st += __builtin_amdgcn_exp2f((e[p].get(k) - at) * kLog2e);
        s = s * (double)(m == mt ? 1.0f : __builtin_amdgcn_exp2f((m - mt) * kLog2e)) + (double)st;
        m = mt;
    }
    // The largest key (0: no candidate)
    __device__ __forceinline__ uint64_t best(uint32_t v, uint32_t stride) const {
        const float x = most();
        uint32_t at = 0;
#pragma unroll
        for (int p = kBeamPieces - 1; p >= 0; --p)
#pragma unroll
            for (int k = kBeamVec - 1; k >= 0; --k)
                if (e[p].get(k) == x) at = v + p * stride + k;
        return x > -INFINITY ? beam_key(x, at) : 0;
    }
    // Logits of the wave that may reach `bound`, at most: those of the pieces whose
    // largest does
    __device__ __forceinline__ int reaching(uint64_t bound) const {
        const float low = beam_low(bound);
        int n = 0;
#pragma unroll
        for (int p = 0; p < kBeamPieces; ++p) n += __popcll(__ballot(top[p] >= low));
        return n * kBeamVec;
    }
    // f(key) for every candidate whose key is at least `bound`; a piece whose largest
    // is below it is passed over
    template <typename F>
    __device__ __forceinline__ void passing(uint64_t bound, uint32_t v, uint32_t stride, F f) const {
        const float low = beam_low(bound);
#pragma unroll
        for (int p = 0; p < kBeamPieces; ++p) {
            if (!(top[p] >= low)) continue;
#pragma unroll
            for (int k = 0; k < kBeamVec; ++k) {
                const float x = e[p].get(k);
                if (!(x >= low)) continue;
                const uint64_t key = beam_key(x, v + p * stride + k);
                if (key >= bound) f(key);
            }
        }
    }
};

// Sum and maximum of a wave's lanes.
__device__ __forceinline__ void beam_wave_sum(float& m, double& s) {
    const float mw = wave_max(m);
    s = wave_sum_f64(m == mw ? s : s * (double)__builtin_amdgcn_exp2f((m - mw) * kLog2e));
    m = mw;
}

// The K-th largest of 64 keys in LDS, by counting the larger ones: each of `nw`
// waves (this one is number w) counts among its 64 / nw keys for all 64, into
// larger[64] (zero before).  After a barrier beam_kth reads it: 1 if fewer than K
// are candidates.
__device__ __forceinline__ void beam_count(const uint64_t* keys, int* larger, int w, int nw) {
    const int lane = threadIdx.x & 63, n = 64 / nw;
    const uint64_t mine = keys[lane];
    int c = 0;
#pragma unroll 4
    for (int i = w * n; i < (w + 1) * n; ++i) c += keys[i] > mine;
    atomicAdd(larger + lane, c);
}
__device__ __forceinline__ uint64_t beam_kth(const uint64_t* keys, const int* larger, int K) {
    const int lane = threadIdx.x & 63;
    const uint64_t mine = keys[lane];
    const unsigned long long at = __ballot(mine != 0 && larger[lane] == K - 1);
    return at ? readlane_u64(mine, __builtin_amdgcn_readfirstlane(__ffsll(at) - 1)) : 1;
}

// Threads that count for one of n entries among `threads` of them: a power of
// two of at most 16.
__device__ __forceinline__ int beam_counters(int n, int threads) {
    int tp = 16;
    while (tp > 1 && n * tp > threads) tp >>= 1;
    return tp;
}

// The K largest keys of a slice of one row.  In the first step: the best key of
// each four threads; the K-th best of those 64 is a bound that at least K keys
// reach (each is the best of its own four threads) and that only K of the fours
// can reach, so at most K * 4 * 32 keys pass into the list.  They are ranked by
// counting the larger ones.  Later steps pass what reaches the K-th best so far;
// only where the list would overflow are it and the step ranked again.
// A full sort or a heap per thread would cost several operations per logit; here a
// logit costs its exponential (a quarter of the rate), a subtraction, two products
// or sums and half a maximum, and a piece of eight one comparison with the bound.
// 512 rows of 65537 bf16, 67 MB: 24 us, 2.8 TB/s, bound by those operations (12 vector
// instructions per logit; they are at work in 59% of a busy CU's cycles) and the
// selection of the first step; fp32, 134 MB, 36 us.  Four blocks per CU: the loads of one step are in flight while the
// present one is summed.
template <typename T>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4)))
beam_row_kernel(const T* __restrict__ logits, BeamArgs a) {
    extern __shared__ uint64_t found[];               // cap = K * 128 + K
    __shared__ uint64_t quad[64], kept[kBeamMaxOut];
    __shared__ float wmax[4];
    __shared__ double wsum[4];
    __shared__ int count[2][4], larger64[64], nfound;
    const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int K = a.K, cap = K * 129;
    const int64_t rec = (int64_t)row * a.slices + slice;
    if (a.finished != nullptr && a.finished[row]) return;     // its logits are not read
    const T* x = logits + (int64_t)row * a.ld;
    const int v0 = slice * (int)a.slice_len, v1 = min(v0 + (int)a.slice_len, (int)a.V);   // (V <= 2^24)
    constexpr int kStride = 256 * kBeamVec;
    float m = -INFINITY;
    double s = 0.0;
    uint64_t bound = 0;                                // 0: no step was ranked yet
    int listed = 0;                                    // entries of the list, at most (in every thread)
    if (tid < K) kept[tid] = 0;
    if (tid == 0) nfound = 0;
    auto load = [&](BeamStep<T>& st, int base) __attribute__((always_inline)) {
        if (base + kBeamTile <= v1) {
#pragma unroll
            for (int p = 0; p < kBeamPieces; ++p) st.e[p].load_whole(x, base + p * kStride + tid * kBeamVec);
        } else {
#pragma unroll
            for (int p = 0; p < kBeamPieces; ++p) st.e[p].load(x, base + p * kStride + tid * kBeamVec, v1);
        }
    };
    auto push = [&](uint64_t key) __attribute__((always_inline)) {
        const int at = atomicAdd(&nfound, 1);
        if (at < cap) found[at] = key;                 // (always, in a row without a signalling NaN)
    };
    // the K best of the list to kept, and the list down to them
    auto rank = [&]() {
        __syncthreads();
        const int n = min(nfound, cap), tp = beam_counters(n, 256);
        for (int i = tid / tp; i < n; i += 256 / tp) {
            const uint64_t key = found[i];
            int larger = 0;
            for (int q = tid & (tp - 1); q < n; q += tp) larger += found[q] > key;
            larger = group_sum_int(larger, tp);
            if (larger < K) kept[larger] = key;        // (the tp threads of an entry alike)
        }
        __syncthreads();
        listed = min(n, K);
        if (tid < listed) found[tid] = kept[tid];
        if (tid == 0) nfound = listed;
        bound = max(kept[K - 1], (uint64_t)1);
        __syncthreads();
    };
    BeamStep<T> cur, next;
    load(cur, v0);
    int step = 0;
    for (int base = v0; base < v1; base += kBeamTile, ++step) {
        if (base + kBeamTile < v1) load(next, base + kBeamTile);
        cur.maxima();
        const uint32_t v = (uint32_t)(base + tid * kBeamVec);
        cur.sum(m, s, (int)v, kStride, v1);
        int all = cap + 1;
        if (bound != 0) {
            const int n = cur.reaching(bound);
            if (lane == 0) count[step & 1][wave] = n;
            __syncthreads();
            all = count[step & 1][0] + count[step & 1][1] + count[step & 1][2] + count[step & 1][3];
        }
        const bool full = listed + all > cap;
        uint64_t low = bound;
        if (full) {
            if (step > 0) rank();
            const uint64_t best = group_max_u64(cur.best(v, kStride), 4);
            if ((tid & 3) == 0) quad[tid >> 2] = best;
            if (tid < 64) larger64[tid] = 0;
            __syncthreads();
            beam_count(quad, larger64, wave, 4);
            __syncthreads();
            low = max(beam_kth(quad, larger64, K), bound);
        }
        if (all > 0) cur.passing(low, v, kStride, push);
        listed += all;
        if (full || base + kBeamTile >= v1) rank();
        cur = next;
    }
    // the slice's sum: threads, then waves
    beam_wave_sum(m, s);
    if (lane == 0) {
        wmax[wave] = m;
        wsum[wave] = s;
    }
    __syncthreads();
    if (tid == 0) {
        const float mb = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
        double sb = 0.0;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            sb += wmax[w] == mb ? wsum[w] : wsum[w] * (double)__builtin_amdgcn_exp2f((wmax[w] - mb) * kLog2e);
        a.part_m[rec] = mb;
        a.part_s[rec] = sb;
    }
    if (tid < K) {
        const uint64_t key = kept[tid];
        a.cand_x[rec * K + tid] = key ? beam_key_x(key) : 0.0f;
        a.cand_v[rec * K + tid] = key ? (int32_t)(uint32_t)~(uint32_t)key : -1;
    }
}

// ------------------------------------------------------------------ groups

struct __align__(16) BeamCand {
    double value;
    uint32_t place;             // (row in group) * V + token; kBeamNone: no candidate
    uint32_t pad;
};
constexpr uint32_t kBeamNone = 0xffffffffu;
// larger value first, then the lower place (a place that is none has value -inf)
__device__ __forceinline__ bool beam_before(const BeamCand& a, const BeamCand& b) {
    return a.value > b.value || (a.value == b.value && a.place < b.place);
}

// A row's candidate as it enters the group: its value and place, or none where
// the value is not finite (a score or a sum that is not; a logit that is ruled out).
__device__ __forceinline__ BeamCand beam_cand(bool any, float x, double lse, float score, int w, int64_t V,
                                              int64_t token) {
    BeamCand c{-INFINITY, kBeamNone, 0};
    const double value = ((double)x - lse) + (double)score;
    if (any && value > -INFINITY && value < INFINITY) {
        c.value = value;
        c.place = (uint32_t)(w * V + token);
    }
    return c;
}

// The best K of n entries of `list` (LDS), `valid` of them candidates, to the
// group's outputs, and the places behind the last candidate; all threads of the
// block, after a barrier.
__device__ __forceinline__ void beam_write(const BeamArgs& a, const BeamCand* list, int n, int valid, int g,
                                           const uint8_t* fin) {
    const int K = a.K, NT = blockDim.x, tid = threadIdx.x, tp = beam_counters(n, NT);
    for (int i = tid / tp; i < n; i += NT / tp) {
        const BeamCand c = list[i];
        if (c.place == kBeamNone) continue;
        int before = 0;
        for (int q = tid & (tp - 1); q < n; q += tp) before += beam_before(list[q], c);
        before = group_sum_int(before, tp);
        if (before >= K || (tid & (tp - 1)) != 0) continue;
        const int64_t o = (int64_t)g * K + before;
        const int w = (int)(c.place / (uint32_t)a.V);
        const int64_t tok = c.place - (int64_t)w * a.V;
        a.out_scores[o] = (float)c.value;
        a.out_parent[o] = g * a.W + w;
        a.out_token[o] = tok;
        if (a.out_finished != nullptr) a.out_finished[o] = fin[w] || tok == a.eos;
    }
    // fewer candidates than places: no parent but the group's first row
    for (int k = valid + tid; k < K; k += NT) {
        const int64_t o = (int64_t)g * K + k;
        a.out_scores[o] = -INFINITY;
        a.out_parent[o] = g * a.W;
        a.out_token[o] = a.pad;
        if (a.out_finished != nullptr) a.out_finished[o] = 0;
    }
}

// One block per group: the rows' sums from their slices', the survivors' values,
// and the K best of them.  More than 256 survivors pass a bound first, as in
// beam_row_kernel: the K-th best of the 64 bests of 16 threads each.  Bound by the
// chain of loads, logarithm, bound and ranking: 64 groups of 8 beams, 5.6 us.
__global__ void __launch_bounds__(1024)
beam_group_kernel(BeamArgs a) {
    __shared__ BeamCand list[kBeamMaxCand], top[64];
    __shared__ double lse[kBeamMaxBeams];
    __shared__ float sc[kBeamMaxBeams];
    __shared__ uint8_t fin[kBeamMaxBeams];
    __shared__ int nfound, larger64[64];
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int W = a.W, K = a.K, S = a.slices, SK = S * K, n = W * SK;
    // the survivors' logits are on their way while the sums are joined
    float cx[2];
    int32_t cv[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = tid + 1024 * k;
        cx[k] = 0.0f;
        cv[k] = -1;
        if (i < n) {
            const int64_t r = (int64_t)g * n + i;
            cx[k] = a.cand_x[r];
            cv[k] = a.cand_v[r];
        }
    }
    if (tid < W) {
        fin[tid] = a.finished != nullptr && a.finished[g * W + tid];
        sc[tid] = a.scores[g * W + tid];
    }
    if (tid == 0) nfound = 0;
    if (tid < 64) larger64[tid] = 0;
    for (int w = wave; w < W; w += 16) {
        const int64_t r = (int64_t)(g * W + w) * S;
        float mb = -INFINITY;
        for (int i = lane; i < S; i += 64) mb = fmaxf(mb, a.part_m[r + i]);
        mb = wave_max(mb);
        double l = 0.0;
        for (int i = lane; i < S; i += 64) {
            const float mi = a.part_m[r + i];
            l += mi == mb ? a.part_s[r + i] : a.part_s[r + i] * exp((double)mi - (double)mb);
        }
        l = wave_sum_f64(l);
        if (lane == 0) lse[w] = (double)mb + log(l);   // -inf: no logit; NaN: a NaN or +inf among them
    }
    __syncthreads();
    BeamCand c[2], best{-INFINITY, kBeamNone, 0};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = tid + 1024 * k, w = i < n ? i / SK : 0;
        const bool f = fin[w];                          // one candidate, its own score
        c[k] = f ? beam_cand(i < n && i - w * SK == 0, 0.0f, 0.0, sc[w], w, a.V, a.pad)
                 : beam_cand(i < n && cv[k] >= 0, cx[k], lse[w], sc[w], w, a.V, cv[k]);
        if (beam_before(c[k], best)) best = c[k];
    }
    BeamCand bound{-INFINITY, kBeamNone, 0};
    if (n > 256) {
        auto better = [&](double v, int p) __attribute__((always_inline)) {
            const BeamCand o{v, (uint32_t)p, 0};
            if (beam_before(o, best)) best = o;
        };
        better(dpp_f64<kDppQuad1032>(best.value), dpp_i32<kDppQuad1032>((int)best.place));
        better(dpp_f64<kDppQuad2301>(best.value), dpp_i32<kDppQuad2301>((int)best.place));
        better(dpp_f64<kDppHalfMirror>(best.value), dpp_i32<kDppHalfMirror>((int)best.place));
        better(dpp_f64<kDppMirror>(best.value), dpp_i32<kDppMirror>((int)best.place));
        if ((tid & 15) == 0) top[tid >> 4] = best;
        __syncthreads();
        // each wave counts among four of the 64 for all of them
        const BeamCand mine = top[lane];
        int before = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) before += beam_before(top[4 * wave + i], mine);
        atomicAdd(larger64 + lane, before);
        __syncthreads();
        const unsigned long long at = __ballot(mine.place != kBeamNone && larger64[lane] == K - 1);
        if (at) bound = top[__builtin_amdgcn_readfirstlane(__ffsll(at) - 1)];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (c[k].place != kBeamNone && !beam_before(bound, c[k])) list[atomicAdd(&nfound, 1)] = c[k];
    __syncthreads();
    beam_write(a, list, nfound, nfound, g, fin);
}

// ------------------------------------------------------------------ a whole group in one block

// Groups of up to kBeamWhole logits (W rounded up to a power of two, times V):
// 16 >> wl waves per row, 32 logits per thread, one launch.  A row's bound comes
// from the bests of 64 equal parts of its threads, so that up to K * (16 >> wl) * 32
// keys pass; ranked, its K best enter the group.  Bound by the latency of that
// chain.  One launch / the two above, in us: 4 beams of 8192 fp32 9.7 / 10.9, 16
// groups of 4 of 4096 bf16 9.3 / 9.9, 1 of 30000 7.4 / 9.0; the host's share of a
// second launch and of a workspace comes on top (2 us).
template <typename T>
__global__ void __launch_bounds__(1024)
beam_whole_kernel(const T* __restrict__ logits, BeamArgs a, int wl, int cap) {
    extern __shared__ uint64_t found[];               // cap per row of the power of two
    __shared__ uint64_t part[kBeamWholeBeams * 64];
    __shared__ BeamCand list[kBeamWholeBeams * kBeamWholeOut];
    __shared__ float wmax[16];
    __shared__ double wsum[16];
    __shared__ int larger[kBeamWholeBeams * 64];
    __shared__ double lse_of[kBeamWholeBeams];
    __shared__ int nfound[kBeamWholeBeams];
    __shared__ uint8_t fin[kBeamWholeBeams];
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int W = a.W, K = a.K, wpr = 16 >> wl;
    const int w = wave >> (4 - wl), sub = wave & (wpr - 1), t = sub * 64 + lane, nt = wpr * 64;   // thread t of nt of row w
    const int row = g * W + min(w, W - 1);
    const bool dead = w >= W, fn = a.finished != nullptr && a.finished[row] != 0;
    const float score = a.scores[row];
    const T* x = logits + (int64_t)row * a.ld;
    const int v1 = dead || fn ? 0 : (int)a.V;          // a finished row's logits are not read
    const int stride = nt * kBeamVec, v = t * kBeamVec;
    BeamStep<T> st;
#pragma unroll
    for (int p = 0; p < kBeamPieces; ++p) st.e[p].load(x, v + p * stride, v1);
    if (t == 0 && !dead) fin[w] = fn;
    if (tid < kBeamWholeBeams) nfound[tid] = 0;
    larger[tid] = 0;                                  // (16 rows of 64: one for each thread)
    float m = -INFINITY;
    double s = 0.0;
    st.maxima();
    st.sum(m, s, v, stride, v1);
    beam_wave_sum(m, s);
    if (lane == 0) {
        wmax[wave] = m;
        wsum[wave] = s;
    }
    const uint64_t best = group_max_u64(st.best((uint32_t)v, (uint32_t)stride), wpr);
    if ((t & (wpr - 1)) == 0) part[w * 64 + t / wpr] = best;
    for (int i = t; i < K; i += nt) list[w * K + i] = BeamCand{-INFINITY, kBeamNone, 0};
    __syncthreads();
    // the row's waves count for the bound; one of them joins the row's sum
    beam_count(part + w * 64, larger + w * 64, sub, wpr);
    if (sub == wpr - 1) {
        const float mi = lane < wpr ? wmax[w * wpr + lane] : -INFINITY, mb = wave_max(mi);
        double l = lane < wpr ? wsum[w * wpr + lane] : 0.0;
        l = wave_sum_f64(mi == mb ? l : l * exp((double)mi - (double)mb));
        if (lane == 0) lse_of[w] = (double)mb + log(l);
    }
    __syncthreads();
    uint64_t* mine = found + (size_t)w * cap;
    st.passing(beam_kth(part + w * 64, larger + w * 64, K), (uint32_t)v, (uint32_t)stride,
               [&](uint64_t key) __attribute__((always_inline)) {
                   const int at = atomicAdd(&nfound[w], 1);
                   if (at < cap) mine[at] = key;       // (always, in a row without a signalling NaN)
               });
    const double lse = lse_of[w];
    __syncthreads();
    const int n = min(nfound[w], cap);
    const int tp = beam_counters(n, nt);
    for (int i = t / tp; i < n; i += nt / tp) {
        const uint64_t key = mine[i];
        int above = 0;
        for (int q = t & (tp - 1); q < n; q += tp) above += mine[q] > key;
        above = group_sum_int(above, tp);
        if (above < K && (t & (tp - 1)) == 0)
            list[w * K + above] = beam_cand(true, beam_key_x(key), lse, score, w, a.V, (uint32_t)~(uint32_t)key);
    }
    if (fn && !dead && t == 0) list[w * K] = beam_cand(true, 0.0f, 0.0, score, w, a.V, a.pad);
    __syncthreads();
    const int valid = __syncthreads_count(tid < W * K && list[tid].place != kBeamNone);    // (at most 512)
    beam_write(a, list, W * K, valid, g, fin);
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
// Rows that stay, and rows whose parent is no row, are not touched: the block
// first lists the rows that move.  Bound by the copy where there is much of it: 256
// rows of 6 tensors, 50 MB read and written, 10 us (a large copy: 9.6); 4 rows 3.6 us,
// a launch and two loads that depend on each other.
template <typename V, int RPT, int NT>
__device__ __forceinline__ void reorder_slice(const ReorderSeg& s, const int2* moves, int n, int tx_log, int slice,
                                              int64_t outer) {
    const int TX = 1 << tx_log, TY = NT >> tx_log;
    const int tx = threadIdx.x & (TX - 1), ty = threadIdx.x >> tx_log;
    const int64_t col = ((int64_t)slice * TX + tx) * sizeof(V);
    char* base = s.p + outer * s.outer_stride + col;
    const bool in = col < s.row_bytes;
    V val[RPT];
    if (in) {
#pragma unroll
        for (int k = 0; k < RPT; ++k)
            if (ty + k * TY < n) val[k] = *reinterpret_cast<const V*>(base + moves[ty + k * TY].y * s.row_stride);
    }
    __syncthreads();
    if (in) {
#pragma unroll
        for (int k = 0; k < RPT; ++k)
            if (ty + k * TY < n) *reinterpret_cast<V*>(base + moves[ty + k * TY].x * s.row_stride) = val[k];
    }
}

template <int RPT, int NT>
__global__ void __launch_bounds__(NT)
reorder_rows_kernel(ReorderArgs a) {
    __shared__ int2 moves[kReorderRows];
    __shared__ int counts[NT / 64];
    int i = 0;
    while (i + 1 < a.nseg && (int)blockIdx.x >= a.seg[i + 1].block0) ++i;
    const ReorderSeg& s = a.seg[i];
    const int k = blockIdx.x - s.block0;
    const int slice = k % s.slices;
    const int64_t outer = k / s.slices;
    const int tid = threadIdx.x, wave = tid >> 6;     // (at most NT rows)
    const int p = tid < a.R ? a.parent[tid] : -1;
    const bool move = p >= 0 && p < a.R && p != tid;
    const unsigned long long who = __ballot(move);
    if ((tid & 63) == 0) counts[wave] = __popcll(who);
    __syncthreads();
    int at = __popcll(who & ((1ull << (tid & 63)) - 1)), n = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        if (w < wave) at += counts[w];
        n += counts[w];
    }
    if (move) moves[at] = make_int2(tid, p);
    __syncthreads();
    if (n == 0) return;
    if (s.vec == 16) reorder_slice<u32x4, RPT, NT>(s, moves, n, a.tx_log, slice, outer);
    else if (s.vec == 4) reorder_slice<uint32_t, RPT, NT>(s, moves, n, a.tx_log, slice, outer);
    else reorder_slice<uint8_t, RPT, NT>(s, moves, n, a.tx_log, slice, outer);
}

// ------------------------------------------------------------------ host side

// Whether one block takes a whole group: the beams' power of two (its logarithm),
// or -1.
static int beam_whole(int64_t W, int64_t V, int64_t K) {
    if (W > kBeamWholeBeams || K > kBeamWholeOut) return -1;
    int wl = 0;
    while ((1 << wl) < W) ++wl;
    return (V << wl) <= kBeamWhole ? wl : -1;
}

// Slices of a row: four blocks per CU (as many as it holds) as long as a slice has
// a step's logits, two per CU down to a quarter of that, and few enough that a
// group's survivors fit one block.  In us with the first number two, four, eight per
// CU: 512 rows of 65537 bf16 37.5, 30.0, 37.7, fp32 45.3, 41.7, 44.2; slices of half a
// step or of a whole one: 512 rows of 8192 13.4, 11.1, 64 rows of 65537 13.7, 13.6.
static int64_t beam_slices(int64_t rows, int64_t W, int64_t V, int64_t K) {
    const int64_t cus = device_cus(), fit = kBeamMaxCand / (W * K);
    int64_t s = ceil_div(4 * cus, rows), least = ceil_div(2 * cus, rows);
    const int64_t full = ceil_div(V, kBeamTile), quarter = ceil_div(V, kBeamTile / 4);
    s = s < full ? s : full;
    least = least < quarter ? least : quarter;
    s = s > least ? s : least;
    s = s < fit ? s : fit;
    return s < 1 ? 1 : s;
}

}  // namespace loom

using namespace loom;

extern "C" int64_t loom_beam_select_workspace_bytes(int64_t groups, int64_t beams, int64_t V, int64_t n_out) {
    if (groups <= 0 || beams <= 0 || V <= 0 || n_out <= 0 || beam_whole(beams, V, n_out) >= 0) return 0;
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
    const int wl = beam_whole(beams, V, n_out);
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
    a.eos = eos_id;
    a.pad = pad_id;
    hipStream_t st = (hipStream_t)stream;
    if (wl >= 0) {
        // (at most K of a row's 64 parts reach its bound, each of (16 >> wl) * 32 logits)
        const int cap = (int)n_out * (16 >> wl) * 32;
        const unsigned lds = (unsigned)((size_t)cap * beams * sizeof(uint64_t));
#define LOOM_BEAM_WHOLE(T) \
        hipLaunchKernelGGL((beam_whole_kernel<T>), dim3((unsigned)groups), dim3(1024), lds, st, (const T*)logits, a, wl, cap)
        if (dtype == LOOM_F32) LOOM_BEAM_WHOLE(float);
        else if (dtype == LOOM_BF16) LOOM_BEAM_WHOLE(bf16_t);
        else LOOM_BEAM_WHOLE(f16_t);
#undef LOOM_BEAM_WHOLE
        return launch_status("loom_beam_select");
    }
    const int64_t rows = groups * beams, S = beam_slices(rows, beams, V, n_out), recs = rows * S;
    a.slice_len = ceil_div(ceil_div(V, S), kBeamVec) * kBeamVec;
    a.slices = (int)S;
    a.part_s = (double*)workspace;
    a.part_m = (float*)(a.part_s + recs);
    a.cand_x = a.part_m + recs;
    a.cand_v = (int32_t*)(a.cand_x + recs * n_out);
    const dim3 grid((unsigned)S, (unsigned)rows);
    const unsigned lds = (unsigned)((n_out * 128 + n_out) * sizeof(uint64_t));
    if (dtype == LOOM_F32)
        hipLaunchKernelGGL((beam_row_kernel<float>), grid, dim3(256), lds, st, (const float*)logits, a);
    else if (dtype == LOOM_BF16)
        hipLaunchKernelGGL((beam_row_kernel<bf16_t>), grid, dim3(256), lds, st, (const bf16_t*)logits, a);
    else
        hipLaunchKernelGGL((beam_row_kernel<f16_t>), grid, dim3(256), lds, st, (const f16_t*)logits, a);
    if (int rc = launch_status("loom_beam_select(rows)")) return rc;
    hipLaunchKernelGGL(beam_group_kernel, dim3((unsigned)groups), dim3(1024), 0, st, a);
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
    // threads across a slice: as many rows at once as there are, at least 16 across (a
    // load of 256 bytes); up to 256 rows in blocks of four waves, RPT rows per thread
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
        const int64_t slices = ceil_div(row_bytes[i], (int64_t)s.vec * tx), most = ((int64_t)1 << 31) - 1 - blocks;
        LOOM_CHECK(slices <= most && outer[i] <= most / slices, "%s: too much data for one call", who);
        s.slices = (int)slices;
        s.block0 = (int)blocks;
        blocks += slices * outer[i];
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
