// select_logprobs.cu -- log-probabilities of given tokens, with entropy, rank and top alternatives.
//
// With y = x / T over a row's n_vocab logits, m = max y, S = sum exp(y - m), A = sum exp(y - m)(y - m):
//   lse = m + ln S,   log p(t) = (y_t - m) - ln S,   H = ln S - A / S,
//   rank(t) = number of ids ahead of t in the order (x descending, id ascending),
//   alternatives = the first n_top ids of that order with their log-probabilities.
// One pass over the logits: each thread keeps (m, S, A) of its elements and rescales S and A when its
// maximum rises (A moves with m: sum e^(y - M)(y - M) = f (A + (m - M) S), f = e^(m - M)). Everything is
// held in f32: A <= 0 <= ln S, so H has no cancellation, and a thread adds at most a few thousand terms.
// Bound: HBM (each logit read once).
//
// Alternatives: each warp keeps the best 32 of its elements as 64-bit rank keys (value, then lower id),
// one per lane, sorted. Few elements get as far as the list: a lane compares the maximum of its elements
// with a threshold that at least n_top elements of the row reach -- the smallest, over the block's
// warps, of their lists' ceil(n_top / warps)-th values, seeded from the first elements' lane maxima.
#include <cfloat>
#include <cmath>
#include <cooperative_groups.h>
#include <cstdint>
#include <cuda_runtime.h>

#include "loom_select.h"
#include "select_device.cuh"
#include "select_internal.h"
#include "select_rows.cuh"

namespace cg = cooperative_groups;

namespace loom_select {
namespace {

constexpr int kLpWarps = 8;
constexpr int kLpNT = kLpWarps * 32;
constexpr int64_t kMaxVocab = int64_t(1) << 30;  // ids, and steps past the last one, in 32 bits
constexpr int kMaxTop = LOOM_SELECT_MAX_TOP_LOGPROBS;
static_assert(kMaxTop <= 32, "a warp's list is one key per lane");
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Exponents are clamped here: 2^-200 is zero in f32, and zero times this is zero (a -inf logit would
// otherwise add 0 * -inf to A).
constexpr float kMinExp2 = -200.0f;

__device__ __forceinline__ float neg_inf() { return -__int_as_float(0x7f800000); }
__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7fc00000); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// max(a, b), NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Softmax state of some elements: reference m (their maximum, at least -FLT_MAX), s = sum 2^((x - m) c)
// and a = sum 2^((x - m) c) (x - m) c. Starting at -FLT_MAX, an all -inf set keeps s = 0.
struct SoftAcc {
    float m, s, a;
};

__device__ __forceinline__ SoftAcc soft_init() { return {-FLT_MAX, 0.0f, 0.0f}; }

// The state moved to reference M >= m.
__device__ __forceinline__ SoftAcc soft_move(SoftAcc p, float M, float c) {
    const float d = fmaxf(__fmul_rn(__fsub_rn(p.m, M), c), kMinExp2);
    const float f = ex2(d);
    return {M, p.s * f, f * __fmaf_rn(d, p.s, p.a)};
}

struct LpDev {
    const unsigned char* base;
    int32_t width;
    int64_t row_stride;
    const int32_t* ids;
    float T, c;
    int32_t n_top;
    float* out_logp;
    float* out_entropy;
    float* out_lse;
    int32_t* out_rank;
    int32_t* out_top_ids;
    float* out_top_logp;
};

struct LpShared {
    SoftAcc acc[kLpWarps];
    int32_t ahead[kLpWarps];
    uint64_t list[kLpWarps][32];
    uint32_t wq[kLpWarps];  // per warp: order key of a value that ceil(n_top / warps) of its elements reach
    // the block's results, read by the cluster's first block
    SoftAcc block_acc;
    int32_t block_ahead;
    uint64_t block_list[32];
};

// Descending bitonic sort of one float per lane.
__device__ __forceinline__ float sort_desc(float v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            const float o = __shfl_xor_sync(0xffffffffu, v, stride);
            v = (((lane & stride) == 0) == ((lane & size) == 0)) ? fmaxf(v, o) : fminf(v, o);
        }
    }
    return v;
}

// The best 32 of two descending lists (one key per lane each), descending.
__device__ __forceinline__ uint64_t merge_lists(uint64_t a, uint64_t b) {
    const int lane = threadIdx.x & 31;
    const uint64_t r = __shfl_sync(0xffffffffu, b, 31 - lane);
    a = a > r ? a : r;  // the best 32, bitonic
#pragma unroll
    for (int stride = 16; stride > 0; stride >>= 1) {
        const uint64_t o = __shfl_xor_sync(0xffffffffu, a, stride);
        a = ((lane & stride) == 0) == (a > o) ? a : o;
    }
    return a;
}

// The states of the warp's first `n` lanes (a power of two) as one, in every one of them: one rescale per
// lane to the common maximum, then plain sums.
__device__ __forceinline__ SoftAcc soft_reduce(SoftAcc p, int n, float c) {
    float M = p.m;
    for (int o = n >> 1; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    p = soft_move(p, M, c);
    for (int o = n >> 1; o > 0; o >>= 1) {
        p.s += __shfl_xor_sync(0xffffffffu, p.s, o);
        p.a += __shfl_xor_sync(0xffffffffu, p.a, o);
    }
    return p;
}

// One thread's running state over its elements of a row.
struct LpScan {
    SoftAcc acc;
    int32_t ahead;
    uint64_t key;   // this lane's entry of the warp's list
    float own;      // smallest float that an element must reach to enter the warp's own list
};

__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}

// Adds NE elements: x[j] has id id0 + (j / kPer) * step + j % kPer; elements whose id is not in
// [0, limit) hold -inf and are neither counted nor listed. All lanes of the warp call it together.
template <int NE, int kPer, bool kTop>
__device__ __forceinline__ void scan_elems(const LpDev& p, LpShared* sh, LpScan& st, const float (&x)[NE], int32_t id0,
                                           int32_t step, int32_t limit, float xt, int32_t t, bool rank) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float mx = x[0];
#pragma unroll
    for (int j = 1; j < NE; ++j) mx = fmaxf(mx, x[j]);
    if (mx > st.acc.m) st.acc = soft_move(st.acc, mx, p.c);
    // Two elements per instruction (f32x2); summed apart first: a thread's chain is one addition per
    // call, not one per element.
    const uint64_t mm = pack2(st.acc.m, st.acc.m), cc = pack2(p.c, p.c);
    uint64_t s2 = 0, a2 = 0;
#pragma unroll
    for (int j = 0; j < NE; j += 2) {
        uint64_t d = pack2(x[j], x[j + 1]);
        asm("sub.rn.f32x2 %0, %0, %1;" : "+l"(d) : "l"(mm));
        asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(d) : "l"(cc));
        float d0, d1;
        unpack2(d, d0, d1);
        d0 = max_nan(d0, kMinExp2);
        d1 = max_nan(d1, kMinExp2);
        d = pack2(d0, d1);
        const uint64_t e = pack2(ex2(d0), ex2(d1));
        asm("add.rn.f32x2 %0, %0, %1;" : "+l"(s2) : "l"(e));
        asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a2) : "l"(e), "l"(d));
    }
    float s0, s1, a0, a1;
    unpack2(s2, s0, s1);
    unpack2(a2, a0, a1);
    st.acc.s += s0 + s1;
    st.acc.a += a0 + a1;
    if (rank && mx >= xt) {
#pragma unroll
        for (int j = 0; j < NE; ++j) {
            const int32_t id = id0 + (j / kPer) * step + j % kPer;
            st.ahead += x[j] > xt || (x[j] == xt && id < t && id >= 0 && id < limit);
        }
    }
    if constexpr (kTop) {
        // the row's threshold: what every warp's wq vouches for together
        uint32_t q = 0xffffffffu;
        if (lane < kLpWarps) q = *reinterpret_cast<volatile uint32_t*>(&sh->wq[lane]);
        q = __reduce_min_sync(0xffffffffu, q);
        const float X = fmaxf(order_key_to_float(q), st.own);
        if (__any_sync(0xffffffffu, mx >= X)) {
            uint32_t hits = 0;
#pragma unroll
            for (int j = 0; j < NE; ++j) {
                const int32_t id = id0 + (j / kPer) * step + j % kPer;
                hits |= uint32_t(x[j] >= X && id >= 0 && id < limit) << j;
            }
            while (__any_sync(0xffffffffu, hits != 0)) {
                uint64_t cand = 0;
                if (hits) {
                    const int at = __ffs(hits) - 1;
                    hits &= hits - 1;
                    float v = x[0];
#pragma unroll
                    for (int j = 1; j < NE; ++j) v = j == at ? x[j] : v;
                    cand = loom_rank_key(v, id0 + (at / kPer) * step + at % kPer);
                }
                uint64_t last = __shfl_sync(0xffffffffu, st.key, p.n_top - 1);
                uint32_t b = __ballot_sync(0xffffffffu, cand > last);
                while (b) {
                    const int src = __ffs(b) - 1;
                    b &= b - 1;
                    const uint64_t k = __shfl_sync(0xffffffffu, cand, src);
                    const int pos = __popc(__ballot_sync(0xffffffffu, st.key > k));
                    const uint64_t up = __shfl_up_sync(0xffffffffu, st.key, 1);
                    if (lane == pos) st.key = k;
                    else if (lane > pos) st.key = up;
                }
            }
            // later elements of this warp have higher ids: an equal value cannot displace the last entry
            const uint64_t last = __shfl_sync(0xffffffffu, st.key, p.n_top - 1);
            if (last) st.own = order_key_to_float(uint32_t(last >> 32) + 1);
            const uint64_t qth = __shfl_sync(0xffffffffu, st.key, (p.n_top + kLpWarps - 1) / kLpWarps - 1);
            if (lane == 0 && uint32_t(qth >> 32) > sh->wq[warp])
                *reinterpret_cast<volatile uint32_t*>(&sh->wq[warp]) = uint32_t(qth >> 32);
        }
    }
}

// The first threshold: each warp's ceil(n_top / warps)-th largest lane maximum is reached by that
// many of its elements. Every thread of the block calls it with the maximum of its first elements.
__device__ __forceinline__ void seed_threshold(const LpDev& p, LpShared* sh, float mx) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float v = __shfl_sync(0xffffffffu, sort_desc(mx), (p.n_top + kLpWarps - 1) / kLpWarps - 1);
    if (lane == 0) sh->wq[warp] = loom_order_key(v);
    __syncthreads();
}

// A cluster of blocks per row: block b of C takes every C-th step of kU * kLpNT vectors. Each block
// reduces its share; the cluster's first block reads the others' results from their shared memory.
// No workspace, tickets or waits between clusters.
template <int kDtype, bool kTop>
__global__ void __launch_bounds__(kLpNT) token_logprobs_kernel(const LpDev p) {
    constexpr int kEsz = kDtype == LOOM_SELECT_BF16 ? 2 : 4;
    constexpr int kPer = 16 / kEsz;
    constexpr int kU = 16 / kPer;  // vectors per thread and step: 16 elements
    __shared__ LpShared sh;
    const cg::cluster_group cluster = cg::this_cluster();
    const int C = int(cluster.num_blocks()), rank_in = int(cluster.block_rank());
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / unsigned(C);
    const unsigned char* rowp = p.base + row * p.row_stride * kEsz;
    // the row as 16-byte aligned vectors: vector v holds ids [v kPer - shift, (v + 1) kPer - shift)
    const int32_t shift = int32_t((reinterpret_cast<uintptr_t>(rowp) & 15) / kEsz);
    const int32_t nv = (shift + p.width + kPer - 1) / kPer;
    const int32_t v0 = shift ? 1 : 0;                                                // first vector inside the row
    const int32_t v1 = max((shift + p.width) / kPer, v0);                            // end of those inside it
    const int32_t limit = v1 * kPer - shift;  // (an id past the whole vectors may be inside the row: an edge's)
    const unsigned char* vec = rowp - shift * kEsz;
    const int32_t stride = C * kU * kLpNT;

    uint4 raw[kU];
    auto load = [&](int32_t v) {
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int32_t vu = v + lane + u * kLpNT;
            if (vu < v1) {
                raw[u] = ldg_stream_v4(vec + int64_t(vu) * 16);
            } else {  // -inf throughout
                const uint32_t w = kDtype == LOOM_SELECT_BF16 ? 0xff80ff80u : 0xff800000u;
                raw[u] = make_uint4(w, w, w, w);
            }
        }
    };
    int32_t v = v0 + rank_in * kU * kLpNT + warp * 32;
    load(v);
    const int32_t t = p.ids ? p.ids[row] : -1;
    const bool has = t >= 0 && t < p.width;
    const float xt = has ? load_global_elem<kDtype>(rowp, t) : quiet_nan();
    const bool rank = p.out_rank != nullptr && has;

    LpScan st{soft_init(), 0, 0ull, neg_inf()};
    // vectors that the row only partly fills: the first (lowest ids, added first) and the last
    auto edge = [&](int32_t v, bool there) {
        float x[kPer];
        const int32_t id0 = v * kPer - shift;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int32_t id = id0 + j;
            x[j] = there && id >= 0 && id < p.width ? load_global_elem<kDtype>(rowp, id) : neg_inf();
        }
        scan_elems<kPer, kPer, kTop>(p, &sh, st, x, there ? id0 : -kPer, 0, p.width, xt, t, rank);
    };
    if constexpr (kTop) {
        float mx = neg_inf();
#pragma unroll
        for (int u = 0; u < kU; ++u) mx = fmaxf(mx, vec_max<kDtype>(raw[u]));  // (NaN left out)
        seed_threshold(p, &sh, mx);
    }
    if (warp == 0 && rank_in == 0 && v0 > 0) edge(0, lane == 0);
    while (v < v1) {  // warp-uniform
        float x[16];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            Vec16<kDtype> e;
            e.unpack(raw[u]);
#pragma unroll
            for (int q = 0; q < kPer; ++q) x[u * kPer + q] = e.x[q];
        }
        const int32_t id0 = (v + lane) * kPer - shift;
        v += stride;
        if (v < v1) load(v);  // the next step's loads are in flight while this one is added
        scan_elems<16, kPer, kTop>(p, &sh, st, x, id0, kLpNT * kPer, limit, xt, t, rank);
    }
    // (the last vector's ids are above all others: after every step of its warp)
    if (warp == 0 && rank_in == 0 && v1 < nv && nv - 1 >= v0) edge(nv - 1, lane == 0);

    // warp, block, cluster
    SoftAcc acc = soft_reduce(st.acc, 32, p.c);
    int32_t ahead = __reduce_add_sync(0xffffffffu, st.ahead);
    if (lane == 0) {
        sh.acc[warp] = acc;
        sh.ahead[warp] = ahead;
    }
    uint64_t key = st.key;
    if constexpr (kTop) {
        // lists by halves: warp w takes in warp w + n's
#pragma unroll
        for (int n = kLpWarps / 2; n > 0; n >>= 1) {
            if (warp >= n && warp < 2 * n) sh.list[warp][lane] = key;
            __syncthreads();
            if (warp < n) key = merge_lists(key, sh.list[warp + n][lane]);
        }
    } else {
        __syncthreads();
    }
    if (warp == 0) {
        acc = lane < kLpWarps ? sh.acc[lane] : soft_init();
        acc = soft_reduce(acc, 32, p.c);
        ahead = __reduce_add_sync(0xffffffffu, lane < kLpWarps ? sh.ahead[lane] : 0);
    }
    if (C > 1) {
        if (warp == 0) {
            if (lane == 0) {
                sh.block_acc = acc;
                sh.block_ahead = ahead;
            }
            if constexpr (kTop) sh.block_list[lane] = key;
        }
        cluster.sync();
        if (rank_in == 0) {
            if constexpr (kTop) {
                // (C is at most kLpWarps: warp b takes block b's list)
                if (warp < C) key = cluster.map_shared_rank(&sh, warp)->block_list[lane];
                for (int n = C / 2; n > 0; n >>= 1) {
                    if (warp >= n && warp < 2 * n) sh.list[warp][lane] = key;
                    __syncthreads();
                    if (warp < n) key = merge_lists(key, sh.list[warp + n][lane]);
                }
            }
            if (warp == 0) {
                acc = soft_init();
                ahead = 0;
                if (lane < C) {
                    const LpShared* other = cluster.map_shared_rank(&sh, lane);
                    acc = other->block_acc;
                    ahead = other->block_ahead;
                }
                acc = soft_reduce(acc, 32, p.c);
                ahead = __reduce_add_sync(0xffffffffu, ahead);
            }
        }
        cluster.sync();  // no block's shared memory goes away before it has been read
    }
    if (warp != 0 || rank_in != 0) return;

    const float lns = logf(acc.s);  // -inf for an empty row, NaN where a logit was NaN or +inf
    const bool empty = acc.s == 0.0f;
    if (lane == 0) {
        const float lse = empty ? neg_inf() : __fdiv_rn(acc.m, p.T) + lns;
        if (p.out_lse) p.out_lse[row] = lse;
        if (p.out_entropy) p.out_entropy[row] = empty ? quiet_nan() : lns - kLn2 * __fdiv_rn(acc.a, acc.s);
        if (p.out_logp) {
            float lp = __fdiv_rn(__fsub_rn(xt, acc.m), p.T) - lns;
            if (empty || (!has && t >= 0)) lp = quiet_nan();
            p.out_logp[row] = t < 0 ? 0.0f : lp;
        }
        if (p.out_rank) p.out_rank[row] = has && xt == xt ? ahead : -1;
    }
    if constexpr (kTop) {
        if (lane < p.n_top) {
            const float v = rank_key_value(key);
            if (p.out_top_ids) p.out_top_ids[row * p.n_top + lane] = key ? rank_key_id(key) : -1;
            if (p.out_top_logp)
                p.out_top_logp[row * p.n_top + lane] =
                    empty || !key ? quiet_nan() : __fdiv_rn(__fsub_rn(v, acc.m), p.T) - lns;
        }
    }
}

// Blocks per row: as many as it takes to fill the GPU (kLpBlocksPerSm resident blocks each), at most 8 (a portable
// cluster), and no more than there are steps of 16 elements a thread in a row.
constexpr int kLpBlocksPerSm = 4;
int lp_cluster(int64_t rows, int64_t n_vocab, int sms) {
    int c = 1;
    while (c < 8 && rows * c < int64_t(kLpBlocksPerSm) * sms && n_vocab > int64_t(c) * 16 * kLpNT) c *= 2;
    return c;
}

template <int kDtype, bool kTop>
cudaError_t launch_lp(const LpDev& p, int64_t rows, int C, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(rows * C));
    cfg.blockDim = dim3(kLpNT);
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = unsigned(C);
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<kDtype, kTop>, p);
}

// ---- the gradient ----
//
// L = sum_r g_r log p_r(t_r) + h_r H_r. With l_j = y_j - lse and p_j = e^(l_j):
//   dL/dx_j = (1/T) [ g (delta_jt - p_j) - h p_j (l_j + H) ]   (dH/dy_j = -p_j (l_j + H)).
// Elementwise once lse and H are there (the forward pass returns them): reads the logits and writes
// the gradient, nothing else. Bound: HBM.
struct LpGradDev {
    const unsigned char* base;
    int64_t width, row_stride;
    const int32_t* ids;
    float inv_t, inv_t_lo;  // 1 / T and what rounding it lost
    const float* lse;
    const float* entropy;
    const float* g_logp;
    const float* g_entropy;
    unsigned char* out;
    int64_t out_stride;
};

template <int kDtype>
__device__ __forceinline__ void store_elem(void* base, int64_t i, float v) {
    if constexpr (kDtype == LOOM_SELECT_BF16) reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<float*>(base)[i] = v;
}

struct LpGradRow {
    float g, h, lse, ent, inv_t, inv_t_lo;
    // x / T - lse with 1 / T in two parts: the rounding of 1 / T alone would be off by |y| 2^-24.
    __device__ __forceinline__ float grad(float x, bool at) const {
        // (-inf logits as -FLT_MAX: their p is 0 all the same, and -inf * 0 would be NaN)
        x = max_nan(x, -FLT_MAX);
        const float l = __fmaf_rn(x, inv_t, __fmaf_rn(x, inv_t_lo, -lse));
        const float e = ex2(__fmul_rn(l, kLog2e));
        float d = e == 0.0f ? 0.0f : -e * (g + (h == 0.0f ? 0.0f : h * (l + ent)));
        if (at) d += g;
        return d * inv_t;
    }
};

constexpr int kGradNT = 256;

template <int kDtype>
__global__ void __launch_bounds__(kGradNT) token_logprobs_grad_kernel(const LpGradDev p) {
    constexpr int kEsz = kDtype == LOOM_SELECT_BF16 ? 2 : 4;
    const int64_t row = blockIdx.x;
    const unsigned char* in = p.base + row * p.row_stride * kEsz;
    unsigned char* out = p.out + row * p.out_stride * kEsz;
    const int64_t t = p.ids ? p.ids[row] : -1;
    LpGradRow r;
    r.g = p.g_logp && t >= 0 ? p.g_logp[row] : 0.0f;
    r.h = p.g_entropy ? p.g_entropy[row] : 0.0f;
    const bool zero = r.g == 0.0f && r.h == 0.0f;
    r.lse = p.lse[row];
    r.ent = r.h != 0.0f ? p.entropy[row] : 0.0f;
    // an id past the vocabulary, an empty row, a row with NaN or +inf: NaN throughout
    const bool bad = (t >= p.width && r.g != 0.0f) || !(fabsf(r.lse) <= FLT_MAX);
    r.inv_t = bad ? quiet_nan() : p.inv_t;
    r.inv_t_lo = p.inv_t_lo;
    for (int64_t j = threadIdx.x; j < p.width; j += kGradNT)
        store_elem<kDtype>(out, j, zero ? 0.0f : r.grad(load_global_elem<kDtype>(in, j), j == t));
}

bool dtype_ok(int dtype) { return dtype == LOOM_SELECT_F32 || dtype == LOOM_SELECT_BF16; }
size_t esz_of(int dtype) { return dtype == LOOM_SELECT_BF16 ? 2 : 4; }
bool misaligned(const void* p, size_t a) { return p && reinterpret_cast<uintptr_t>(p) % a != 0; }

// T and log2(e) / T have to be normal numbers.
bool temperature_ok(float T) { return T >= FLT_MIN && T <= FLT_MAX; }

}  // namespace
}  // namespace loom_select

using namespace loom_select;

extern "C" {

LOOM_SELECT_API int loom_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t n_vocab,
                                        int64_t row_stride, const int32_t* ids, float temperature, int32_t n_top,
                                        float* out_logp, float* out_entropy, float* out_lse, int32_t* out_rank,
                                        int32_t* out_top_ids, float* out_top_logp, void* stream) {
    if (!dtype_ok(dtype)) return LOOM_SELECT_EDTYPE;
    if (!logits || rows <= 0 || n_vocab <= 0 || row_stride < n_vocab) return LOOM_SELECT_EINVAL;
    if (!out_logp && !out_entropy && !out_lse && !out_rank && !out_top_ids && !out_top_logp) return LOOM_SELECT_EINVAL;
    if ((out_logp || out_rank) && !ids) return LOOM_SELECT_EINVAL;
    if (misaligned(logits, esz_of(dtype)) || misaligned(ids, 4) || misaligned(out_logp, 4) ||
        misaligned(out_entropy, 4) || misaligned(out_lse, 4) || misaligned(out_rank, 4) ||
        misaligned(out_top_ids, 4) || misaligned(out_top_logp, 4))
        return LOOM_SELECT_EINVAL;
    if (!temperature_ok(temperature)) return LOOM_SELECT_EPARAM;
    if (n_top < 0 || n_top > kMaxTop || n_top > n_vocab) return LOOM_SELECT_EPARAM;
    if ((n_top > 0) != (out_top_ids || out_top_logp)) return LOOM_SELECT_EINVAL;
    if (n_vocab > kMaxVocab || rows > INT32_MAX / 16) return LOOM_SELECT_ESHAPE;
    LpDev p;
    p.base = static_cast<const unsigned char*>(logits);
    p.width = int32_t(n_vocab);
    p.row_stride = row_stride;
    p.ids = ids;
    p.T = temperature;
    p.c = float(1.4426950408889634 / double(temperature));
    p.n_top = n_top;
    p.out_logp = out_logp;
    p.out_entropy = out_entropy;
    p.out_lse = out_lse;
    p.out_rank = out_rank;
    p.out_top_ids = out_top_ids;
    p.out_top_logp = out_top_logp;
    int st = LOOM_SELECT_OK;
    const int sms = device_sm_count(&st);
    if (st != LOOM_SELECT_OK) return st;
    const int C = lp_cluster(rows, n_vocab, sms);
    const auto s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (dtype == LOOM_SELECT_BF16)
        e = n_top ? launch_lp<LOOM_SELECT_BF16, true>(p, rows, C, s) : launch_lp<LOOM_SELECT_BF16, false>(p, rows, C, s);
    else
        e = n_top ? launch_lp<LOOM_SELECT_F32, true>(p, rows, C, s) : launch_lp<LOOM_SELECT_F32, false>(p, rows, C, s);
    return e == cudaSuccess ? LOOM_SELECT_OK : LOOM_SELECT_ECUDA;
}

LOOM_SELECT_API int loom_token_logprobs_grad(const void* logits, int dtype, int64_t rows, int64_t n_vocab,
                                             int64_t row_stride, const int32_t* ids, float temperature,
                                             const float* lse, const float* entropy, const float* grad_logp,
                                             const float* grad_entropy, void* out_grad, int64_t grad_stride,
                                             void* stream) {
    if (!dtype_ok(dtype)) return LOOM_SELECT_EDTYPE;
    if (!logits || !lse || !out_grad || rows <= 0 || n_vocab <= 0 || row_stride < n_vocab || grad_stride < n_vocab)
        return LOOM_SELECT_EINVAL;
    if ((!grad_logp && !grad_entropy) || (grad_logp && !ids) || (grad_entropy && !entropy)) return LOOM_SELECT_EINVAL;
    if (misaligned(logits, esz_of(dtype)) || misaligned(out_grad, esz_of(dtype)) || misaligned(ids, 4) ||
        misaligned(lse, 4) || misaligned(entropy, 4) || misaligned(grad_logp, 4) || misaligned(grad_entropy, 4))
        return LOOM_SELECT_EINVAL;
    if (!temperature_ok(temperature)) return LOOM_SELECT_EPARAM;
    if (n_vocab > kMaxVocab || rows > INT32_MAX / 16) return LOOM_SELECT_ESHAPE;
    // in place only element for element
    if (logits == out_grad && row_stride != grad_stride) return LOOM_SELECT_EINVAL;
    LpGradDev p;
    p.base = static_cast<const unsigned char*>(logits);
    p.width = n_vocab;
    p.row_stride = row_stride;
    p.ids = ids;
    const double inv = 1.0 / double(temperature);
    p.inv_t = float(inv);
    p.inv_t_lo = float(inv - double(p.inv_t));
    p.lse = lse;
    p.entropy = entropy;
    p.g_logp = grad_logp;
    p.g_entropy = grad_entropy;
    p.out = static_cast<unsigned char*>(out_grad);
    p.out_stride = grad_stride;
    const auto s = static_cast<cudaStream_t>(stream);
    if (dtype == LOOM_SELECT_BF16) token_logprobs_grad_kernel<LOOM_SELECT_BF16><<<unsigned(rows), kGradNT, 0, s>>>(p);
    else token_logprobs_grad_kernel<LOOM_SELECT_F32><<<unsigned(rows), kGradNT, 0, s>>>(p);
    return cudaGetLastError() == cudaSuccess ? LOOM_SELECT_OK : LOOM_SELECT_ECUDA;
}

}  // extern "C"
