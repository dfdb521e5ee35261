// select_logprobs.cu -- log-probabilities of given tokens, with entropy, rank and top alternatives.
//
// With y = x / T over a row's n_vocab logits, m = max y, S = sum exp(y - m), A = sum exp(y - m)(y - m):
//   lse = m + ln S,   log p(t) = (y_t - m) - ln S,   H = ln S - A / S
// (S near 1, as ln(1 + (S - 1)) from a sum without the largest element: log p keeps its digits where p is near 1),
//   rank(t) = number of ids ahead of t in the order (x descending, id ascending),
//   alternatives = the first n_top ids of that order with their log-probabilities.
// One pass over the logits: each thread keeps (m, S, A) of its elements and rescales S and A when its
// maximum rises (A moves with m: sum e^(y - M)(y - M) = f (A + (m - M) S), f = e^(m - M)). Everything is
// held in f32: A <= 0 <= ln S, so H has no cancellation, and a thread adds at most a few thousand terms.
// Bound: HBM (each logit read once) for many rows, [1024, 151936] f32 in 100.0 us (6.2 TB/s; 93.5 without rank and
// alternatives); the latency of a row's end, some ten dependent steps, for few: 8.0 us for one row of 151936.
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

constexpr int64_t kMaxVocab = int64_t(1) << 30;  // ids, and steps past the last one, in 32 bits
constexpr int kMaxTop = LOOM_SELECT_MAX_TOP_LOGPROBS;
static_assert(kMaxTop <= 32, "a warp's list is one key per lane");
constexpr float kLn2 = 0.6931471805599453f;
// Exponents are clamped here: 2^-200 is zero in f32, and zero times this is zero (a -inf logit would
// otherwise add 0 * -inf to A).
constexpr float kMinExp2 = -200.0f;

// A row whose sum of exponentials, its largest element's 1 among them, is below this is added up without that one.
constexpr float kNearOne = 1.25f;

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
    int64_t rows;
    int32_t width;
    int64_t row_stride;
    const int32_t* ids;
    float c;                // log2(e) / T
    float inv_t, inv_t_lo;  // 1 / T and what rounding it lost
    int32_t n_top;
    float* out_logp;
    float* out_entropy;
    float* out_lse;
    int32_t* out_rank;
    int32_t* out_top_ids;
    float* out_top_logp;
};

// A thread keeps the maxima of its elements in up to this many equal runs of steps (32: 117.4 us for [1024, 151936] f32,
// 16: 115.1, the shared memory being L1's).
constexpr int kSlots = 16;
static_assert(kSlots <= 32, "a thread's slots are bits of a word");
constexpr int kMaxCluster = 8;
constexpr int kGroups = 64;  // (32 where a row is one warp's)
// Warps to a row: 8 in each block of a cluster, 4 (a block to a row), or 1 (four rows to a block).
constexpr int kLpWarps = 8, kLpRowWarps = 4;

template <int kW, bool kTop>
struct LpShared {
    static constexpr int kMaxCand = !kTop ? 1 : kW == kLpWarps ? 512 : 256;
    static constexpr int kSlotsHere = kTop ? kSlots : 1;
    static constexpr int kBlocks = kW == kLpWarps ? kMaxCluster : 1;
    uint64_t list[kW][32];
    alignas(16) uint32_t group[kGroups];  // order keys of the maxima of the cluster's groups of threads
    uint32_t x_key;            // order key of the threshold
    int32_t n_cand;            // elements of this block that reach it
    int32_t overflow;          // some block of the cluster has more of them than it may hand on
    union {  // (sorted once the slots have been looked through)
        float slot_max[kW][kSlotsHere][32];
        uint64_t sorting[kMaxCand + 8];
    };
    float edge[32];            // the elements apart from the vectors (the first block's)
    // of the cluster's first block: what the blocks hand on
    SoftAcc acc[kBlocks * kW];  // of each warp
    float others[kBlocks * kW];  // its sum without that of the lane with its maximum
    int32_t lead[kBlocks * kW];  // that lane
    int32_t ahead[kBlocks * kW];
    int32_t part_cand[kBlocks];
    float m, lns;              // the row's, from the warp that has them to the one with the alternatives
    uint64_t cand[kMaxCand];   // kMaxCand / C from each block
    uint64_t part_list[kBlocks][32];
};

// Descending bitonic sort of one key per lane.
__device__ __forceinline__ uint64_t sort_desc(uint64_t v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            const uint64_t o = __shfl_xor_sync(0xffffffffu, v, stride);
            v = ((((lane & stride) == 0) == ((lane & size) == 0)) == (v > o)) ? v : o;
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

// Of the warp's states, moved to their common maximum M: the first lane that has it, and the sum of the others' s.
__device__ __forceinline__ float soft_others(SoftAcc p, float M, float c, int32_t& lead) {
    lead = __ffs(__ballot_sync(0xffffffffu, p.m == M && p.s > 0.0f)) - 1;
    float s = int32_t(threadIdx.x & 31) == lead ? 0.0f : soft_move(p, M, c).s;
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}

// 1 where a > b (kGe: a >= b), else 0 (NaN: 0).
template <bool kGe>
__device__ __forceinline__ float ahead_one(float a, float b) {
    float y;
    if constexpr (kGe) asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    else asm("set.gt.f32.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// One 16-byte vector as pairs of floats.
template <int kDtype>
struct Pairs {
    static constexpr int kPairs = kDtype == LOOM_SELECT_BF16 ? 4 : 2;
    uint64_t v[kPairs];
    __device__ __forceinline__ explicit Pairs(uint4 raw) {
        if constexpr (kDtype == LOOM_SELECT_BF16) {
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = pack2(__uint_as_float(w[q] << 16), __uint_as_float(w[q] & 0xffff0000u));
        } else {
            v[0] = pack2(__uint_as_float(raw.x), __uint_as_float(raw.y));
            v[1] = pack2(__uint_as_float(raw.z), __uint_as_float(raw.w));
        }
    }
};

__device__ __forceinline__ void add2(uint64_t& a, uint64_t b) { asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a) : "l"(b)); }
__device__ __forceinline__ void fma2(uint64_t& d, uint64_t a, uint64_t b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(a), "l"(b));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// The largest element of kU vectors (at least -inf; NaN left out).
template <int kDtype, int kU>
__device__ __forceinline__ float largest(const uint4 (&raw)[kU]) {
    if constexpr (kDtype == LOOM_SELECT_BF16) {
        __nv_bfloat162 m = *reinterpret_cast<const __nv_bfloat162*>(&raw[0].x);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (u || q) m = __hmax2(m, *reinterpret_cast<const __nv_bfloat162*>(&w[q]));
        }
        return max3(__low2float(m), __high2float(m), neg_inf());
    } else {
        float m = neg_inf();
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            m = max3(m, __uint_as_float(raw[u].x), __uint_as_float(raw[u].y));
            m = max3(m, __uint_as_float(raw[u].z), __uint_as_float(raw[u].w));
        }
        return m;
    }
}

// One thread's running softmax sums and rank count over its elements of a row, which come as kU vectors of kPer
// elements each: element q of vector u has id id0 + u * step + q; those whose id is not in [0, limit) hold -inf and
// are not counted.
template <int kDtype, int kU>
struct LpScan {
    static constexpr int kPer = kDtype == LOOM_SELECT_BF16 ? 8 : 4;
    SoftAcc acc;
    float c;         // log2(e) / T
    float mc;        // rn(m c)
    bool slow;
    int32_t ahead;

    __device__ __forceinline__ void start(float c_) {
        acc = soft_init();
        c = c_;
        mc = -neg_inf();  // (until there is a maximum, the common path gives NaN)
        slow = false;
        ahead = 0;
    }

    // A maximum above the last one.
    __device__ __forceinline__ void rise(float mx) {
        acc = soft_move(acc, mx, c);
        mc = __fmul_rn(mx, c);
        slow = slow || !(fabsf(mc) <= 65536.0f);
    }

    // One element apart from the vectors.
    __device__ __forceinline__ void add_edge(float x) {
        if (x > acc.m) rise(x);
        add_one(x, acc.s, acc.a);
    }

    // Two elements per instruction (f32x2). The common path takes 2^(x c - rn(m c)), one fused operation, one ex2 and
    // two additions an element, and moves the vectors' sums to the exact reference m c afterwards. A -inf (its
    // product with the exponent is NaN), a NaN, or a maximum so large that rounding m c loses much send the thread
    // to the other path from then on: (x - m) c, clamped. `partial`: some elements are not there.
    __device__ __forceinline__ void add(const uint4 (&raw)[kU], float mx, bool partial) {
        if (mx > acc.m) rise(mx);
        float s, a;
        bool clamped = slow || partial;
        if (!clamped) {
            const uint64_t cc = pack2(c, c), mm = pack2(-mc, -mc);
            uint64_t s2 = 0, a2 = 0;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const Pairs<kDtype> x(raw[u]);
#pragma unroll
                for (int q = 0; q < Pairs<kDtype>::kPairs; ++q) {
                    uint64_t d;
                    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(x.v[q]), "l"(cc), "l"(mm));
                    float d0, d1;
                    unpack2(d, d0, d1);
                    const uint64_t e = pack2(ex2(d0), ex2(d1));
                    add2(s2, e);
                    fma2(a2, e, d);
                }
            }
            float s0, s1, a0, a1;
            unpack2(s2, s0, s1);
            unpack2(a2, a0, a1);
            s = s0 + s1;
            const float r = __fmaf_rn(acc.m, c, -mc), g = ex2(-r);  // what rounding m c lost
            a = __fmaf_rn(-r, s, a0 + a1) * g;
            s *= g;
            clamped = slow = a != a;
        }
        if (clamped) {
            s = a = 0.0f;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const Pairs<kDtype> x(raw[u]);
#pragma unroll
                for (int q = 0; q < Pairs<kDtype>::kPairs; ++q) {
                    float x0, x1;
                    unpack2(x.v[q], x0, x1);
                    add_one(x0, s, a);
                    add_one(x1, s, a);
                }
            }
        }
        acc.s += s;
        acc.a += a;
    }

    __device__ __forceinline__ void add_one(float x, float& s, float& a) const {
        const float d = max_nan(__fmul_rn(__fsub_rn(x, acc.m), c), kMinExp2);
        const float e = ex2(d);
        s += e;
        a = __fmaf_rn(e, d, a);
    }

    // Elements above xt, or (kGe) not below it.
    template <bool kGe>
    __device__ __forceinline__ void count_all(const uint4 (&raw)[kU], float xt) {
        if constexpr (kDtype == LOOM_SELECT_BF16) {
            // packed: at most kU * 4 to a half, exact in bf16
            const __nv_bfloat162 t2 = __float2bfloat162_rn(xt);
            __nv_bfloat162 n = __float2bfloat162_rn(0.0f);
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&w[q]);
                    n = __hadd2(n, kGe ? __hge2(x, t2) : __hgt2(x, t2));
                }
            }
            ahead += int32_t(__low2float(n) + __high2float(n));
        } else {
            uint64_t n2 = 0;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const float x[4] = {__uint_as_float(raw[u].x), __uint_as_float(raw[u].y), __uint_as_float(raw[u].z),
                                    __uint_as_float(raw[u].w)};
                add2(n2, pack2(ahead_one<kGe>(x[0], xt), ahead_one<kGe>(x[1], xt)));
                add2(n2, pack2(ahead_one<kGe>(x[2], xt), ahead_one<kGe>(x[3], xt)));
            }
            float n0, n1;
            unpack2(n2, n0, n1);
            ahead += int32_t(n0 + n1);
        }
    }

    // Ids ahead of t, whose logit is xt: x > xt, or x == xt and a lower id. The warp's ids of this call are in
    // [lo, hi): all before t or all after it, usually.
    __device__ __forceinline__ void count(const uint4 (&raw)[kU], float mx, int32_t id0, int32_t step, int32_t limit,
                                          int32_t lo, int32_t hi, float xt, int32_t t) {
        if (!__any_sync(0xffffffffu, mx >= xt)) return;
        if (lo > t) {
            count_all<false>(raw, xt);
        } else if (hi <= t && xt > neg_inf()) {  // (the -inf of elements that are not there must not count)
            count_all<true>(raw, xt);
        } else {
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                Vec16<kDtype> e;
                e.unpack(raw[u]);
#pragma unroll
                for (int q = 0; q < kPer; ++q) {
                    const int32_t id = id0 + u * step + q;
                    ahead += e.x[q] > xt || (e.x[q] == xt && id < t && id >= 0 && id < limit);
                }
            }
        }
    }
};

// One warp's view of its row, for looking through the slots again.
struct LpShare {
    const unsigned char* row;
    int32_t shift, v_start, v1, stride, per_slot, slots;  // v_start: the warp's first vector
    int n_top;
    float X;
};

// The elements that the lanes in `hits` have in slot `slot` (each lane's own), spread over the warp 32 at a time: f gets
// four values and their ids, NaN where there is none, in all lanes. Four lanes' elements are requested together. A loop with
// little code: unrolled over a thread's own elements, instruction fetches made this 7000 cycles and not 1500.
template <int kDtype, int kU, int kNT, class F>
__device__ __forceinline__ void visit(const LpShare& r, uint32_t hits, int32_t slot, F&& f) {
    constexpr int kPer = kDtype == LOOM_SELECT_BF16 ? 8 : 4;
    const int lane = threadIdx.x & 31;
    while (hits) {
        int32_t first[4];  // of each of four lanes, its first vector in the slot
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int src = __ffs(hits) - 1;
            hits &= hits - 1;  // (0 stays 0)
            const int32_t of = __shfl_sync(0xffffffffu, slot, src < 0 ? 0 : src);
            first[k] = src < 0 ? r.v1 : r.v_start + src + of * r.per_slot * r.stride;
        }
        for (int e0 = 0; e0 < r.per_slot * kU * kPer; e0 += 32) {
            const int e = e0 + lane;
            const int32_t skip = e / (kU * kPer) * r.stride + e / kPer % kU * kNT;
            float x[4];
            int32_t id[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int32_t v = first[k] + skip;
                x[k] = e < r.per_slot * kU * kPer && v < r.v1 ? load_global_elem<kDtype>(r.row, v * kPer - r.shift + e % kPer)
                                                             : quiet_nan();
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) id[k] = (first[k] + skip) * kPer - r.shift + e % kPer;
            f(x, id);
        }
    }
}

// The warp's best 32 of its elements >= X, sorted, when too many of them reach X to be held (a row of few
// values, or of almost nothing but -inf).
template <int kDtype, int kU, int kW>
__device__ __noinline__ uint64_t list_slots(const LpShare& r, LpShared<kW, true>* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32 % kW;
    uint64_t key = 0;
    float own = neg_inf();
    for (int32_t s = 0; s < r.slots; ++s) {
        const uint32_t hits = __ballot_sync(0xffffffffu, sh->slot_max[warp][s][lane] >= fmaxf(r.X, own));
        visit<kDtype, kU, kW * 32>(r, hits, s, [&](const float(&x)[4], const int32_t(&id)[4]) {
#pragma unroll 1
            for (int k = 0; k < 4; ++k) {
                const float xk = k == 0 ? x[0] : k == 1 ? x[1] : k == 2 ? x[2] : x[3];
                const int32_t ik = k == 0 ? id[0] : k == 1 ? id[1] : k == 2 ? id[2] : id[3];
                const uint64_t cand = xk >= r.X ? loom_rank_key(xk, ik) : 0ull;
                if (__any_sync(0xffffffffu, cand > __shfl_sync(0xffffffffu, key, r.n_top - 1)))
                    key = merge_lists(key, sort_desc(cand));
            }
        });
        // a later slot's ids are above all earlier ones: only a larger value can displace the list's last
        const uint64_t last = __shfl_sync(0xffffffffu, key, r.n_top - 1);
        own = last ? order_key_to_float(uint32_t(last >> 32) + 1) : neg_inf();
    }
    return key;
}

// The sum of 2^((x - m) c) over the elements of one lane of the row, whose first vector is v, without its maximum m: read
// again by a whole warp. (In line: as a call it cost one row of 51865 bf16 with 5 alternatives, which does not come here,
// 1.4 us of 7.0.)
template <int kDtype, int kU, int kNT>
__device__ __forceinline__ float sum_without_max(const unsigned char* vec, int32_t v, int32_t v1, int32_t stride, float m, float c) {
    const int lane = threadIdx.x & 31;
    const int32_t n = v < v1 ? ((v1 - v + stride - 1) / stride) * kU : 0;
    float s = 0.0f;
    for (int32_t i0 = 0; i0 < n; i0 += 4 * 32) {
        uint4 raw[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int32_t i = i0 + k * 32 + lane, at = v + i / kU * stride + i % kU * kNT;
            const uint32_t none = kDtype == LOOM_SELECT_BF16 ? 0xff80ff80u : 0xff800000u;
            raw[k] = make_uint4(none, none, none, none);
            if (i < n && at < v1) raw[k] = ldg_stream_v4(vec + int64_t(at) * 16);
        }
#pragma unroll 1
        for (int k = 0; k < 4; ++k) {
            Vec16<kDtype> e;
            e.unpack(k == 0 ? raw[0] : k == 1 ? raw[1] : k == 2 ? raw[2] : raw[3]);
#pragma unroll
            for (int q = 0; q < Vec16<kDtype>::kElems; ++q)
                if (e.x[q] != m) s += ex2(max_nan(__fmul_rn(__fsub_rn(e.x[q], m), c), kMinExp2));
        }
    }
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// Up to this width, and for more than 8 alternatives, the lanes of a row's one warp look through their own slots, of few
// elements and most of them hit ([16384, 1025] f32 with 20 45.3 us when it was measured (47.7 now), by the warp together
// 63.5; [8000, 8000] bf16 70.1 and 65.8; with 5 [700, 2048] f32 8.6 and 7.7).
constexpr int32_t kOwnSlots = 4096;

template <int kW>
__device__ __forceinline__ void block_sync() {
    if constexpr (kW == 1) __syncwarp();
    else __syncthreads();
}

// A cluster of C blocks of kW warps per row: block b takes every C-th step of kU vectors per thread, and hands its
// share's results to the cluster's first block through distributed shared memory. No workspace, tickets or waits
// between clusters.
//
// Alternatives: while streaming, a thread only notes the largest element of each slot (a run of steps). At the end
// the n_top-th largest of 64 maxima, of equal groups of the cluster's threads, is a threshold that at least n_top
// elements of the row reach, and few more do (64 -ln(1 - n / 64): 24 for 20). The slots whose maximum reaches it are
// read again, from L2, and those elements sorted by counting the larger ones.
//
// Blocks of eight warps, in clusters where there are few rows: four to an SM ([256, 262144] bf16 41.5 us, four warps 50.2).
// Where there are rows for all of them, blocks of four take a row each, with a row's end among more rows' streams and less
// lost to the last wave: [1024, 151936] f32 100.0 us (eight warps 111.1, two 150.1), [600, 51864] bf16 25.0 (33.7). Seven of
// them to an SM (72 registers; eight, of 64, 101.1 and 26.9, [3000, 32000] bf16 71.9 where seven take 64.8), and seven of
// four rows a warp each ([8000, 8000] f32 53.6 us, six 62.4).
// kU: vectors per thread and step. Four ([1024, 151936] f32 102.8 us as it then was; three: 106.9, five: 106.1). Eight where
// every block has an SM to itself and two such steps or more to read (then 1 row of 151936 f32 8.4 us, with four 9.6, 18
// rows 10.1 and 10.9; with less to read, one of 51865 bf16 7.8 and 7.3, 18 of 151936 bf16 10.5 and 9.9). Two for a warp's
// row of at most two such steps, eight blocks to an SM ([20000, 300] bf16 without alternatives 15.6 us, with four 21.0;
// [20000, 800] f32 23.5 and 19.9; all of these before rows with a likely id were summed twice).
template <int kDtype, bool kTop, int kW, int kU>
__global__ void __launch_bounds__(kW == 1 ? 128 : kW * 32, kU == 2 ? 8 : kU == 8 ? 2 : kW < 8 ? 7 : 4)
    token_logprobs_kernel(const LpDev p) {
    constexpr int kEsz = kDtype == LOOM_SELECT_BF16 ? 2 : 4;
    constexpr int kPer = 16 / kEsz;
    constexpr int kNT = kW * 32;
    constexpr int kRows = kW == 1 ? 4 : 1;
    __shared__ LpShared<kW, kTop> sh_of_row[kRows];
    LpShared<kW, kTop>& sh = sh_of_row[kW == 1 ? threadIdx.x / 32 : 0];
    const cg::cluster_group cluster = cg::this_cluster();
    const int C = kW == kLpWarps ? int(cluster.num_blocks()) : 1, rank_in = kW == kLpWarps ? int(cluster.block_rank()) : 0;
    const int tid = threadIdx.x % (kW * 32), lane = tid & 31, warp = tid >> 5;
    const int64_t row = kW == 1 ? int64_t(blockIdx.x) * kRows + threadIdx.x / 32 : blockIdx.x / unsigned(C);
    if (kW == 1 && row >= p.rows) return;
    const int32_t t = p.ids ? p.ids[row] : -1;
    const unsigned char* rowp = p.base + row * p.row_stride * kEsz;
    // the row as 16-byte aligned vectors: vector v holds ids [v kPer - shift, (v + 1) kPer - shift)
    const int32_t shift = int32_t((reinterpret_cast<uintptr_t>(rowp) & 15) / kEsz);
    const int32_t nv = (shift + p.width + kPer - 1) / kPer;
    const int32_t v0 = shift ? 1 : 0;                      // first vector inside the row
    const int32_t v1 = max((shift + p.width) / kPer, v0);  // end of those inside it
    const unsigned char* vec = rowp - shift * kEsz;
    const int32_t stride = C * kU * kNT;
    const int32_t steps = (v1 - v0 + stride - 1) / stride;
    const int32_t per_slot = (steps + kSlots - 1) / kSlots;

    // A step's vectors for this lane; in a step that the row's end cuts, those past it are -inf throughout.
    const int32_t v_start = v0 + rank_in * kU * kNT + warp * 32;
    auto whole = [&](int32_t v) { return v + (kU - 1) * kNT + 32 <= v1; };  // (the warp's step at v)
    auto load = [&](uint4(&raw)[kU], int32_t v) {
        const unsigned char* at = vec + int64_t(v + lane) * 16;
        if (whole(v)) {
#pragma unroll
            for (int u = 0; u < kU; ++u) raw[u] = ldg_stream_v4(at + u * kNT * 16);
        } else {
            const uint32_t w = kDtype == LOOM_SELECT_BF16 ? 0xff80ff80u : 0xff800000u;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                raw[u] = make_uint4(w, w, w, w);
                if (v + lane + u * kNT < v1) raw[u] = ldg_stream_v4(at + u * kNT * 16);
            }
        }
    };
    int32_t v = v_start;
    uint4 raw_a[kU], raw_b[kU];  // the step being added and the next one, whose loads are in flight
    if (v < v1) load(raw_a, v);
    // the elements of the vectors that the row only partly fills, at most one to a lane of the cluster's first warp: those
    // of the first in lanes 0 .. kPer - 1, those of the last in kPer .. 2 kPer - 1; -1: none
    auto edge_id = [&] {
        int32_t id = -1;
        if (lane < kPer && v0 > 0) id = lane - shift;
        if (lane >= kPer && lane < 2 * kPer && v1 < nv && nv - 1 >= v0) id = (nv - 1) * kPer - shift + lane - kPer;
        return warp == 0 && rank_in == 0 && id < p.width ? id : -1;
    };
    if (tid == 0) sh.n_cand = sh.overflow = 0;
    if (C > 1) cluster.barrier_arrive();  // (waited for before the first remote store: all blocks have begun)

    LpScan<kDtype, kU> st;
    st.start(p.c);
    const bool has = t >= 0 && t < p.width;
    const float xt = has ? load_global_elem<kDtype>(rowp, t) : quiet_nan();
    const bool rank = p.out_rank != nullptr && has;
    if (warp == 0 && rank_in == 0) {
        const int32_t id = edge_id();
        const float x = id >= 0 ? load_global_elem<kDtype>(rowp, id) : neg_inf();
        st.add_edge(x);
        st.ahead += rank && id >= 0 && (x > xt || (x == xt && id < t));
        sh.edge[lane] = x;
    }

    float slot_top = neg_inf();  // this thread's maximum in the current slot
    float* slot_at = &sh.slot_max[warp][0][lane];
    int32_t left = per_slot;  // steps of that slot to come
    auto step = [&](const uint4(&raw)[kU], int32_t at) {
        const float mx = largest<kDtype>(raw);
        st.add(raw, mx, !whole(at));
        if (rank)
            st.count(raw, mx, (at + lane) * kPer - shift, kNT * kPer, v1 * kPer - shift, at * kPer - shift,
                     (at + (kU - 1) * kNT + 32) * kPer - shift, xt, t);
        if constexpr (kTop) {
            slot_top = fmaxf(slot_top, mx);
            if (--left == 0) {
                *slot_at = slot_top;
                slot_at += 32;
                slot_top = neg_inf();
                left = per_slot;
            }
        }
    };
    while (v < v1) {  // warp-uniform
        if (v + stride < v1) load(raw_b, v + stride);
        step(raw_a, v);
        v += stride;
        if (v >= v1) break;
        if (v + stride < v1) load(raw_a, v + stride);
        step(raw_b, v);
        v += stride;
    }
    if (kTop && left != per_slot) {
        *slot_at = slot_top;
        slot_at += 32;
    }
    LpShared<kW, kTop>* first = C > 1 ? cluster.map_shared_rank(&sh, 0) : &sh;

    // this thread's maximum (none: s is 0, or NaN, as nothing above -FLT_MAX shows)
    const float top = st.acc.m > -FLT_MAX || st.acc.s > 0.0f ? st.acc.m : neg_inf();
    // softmax state and rank of the warp, and the maxima of the groups of threads
    SoftAcc acc = soft_reduce(st.acc, 32, p.c);
    int32_t ahead = __reduce_add_sync(0xffffffffu, st.ahead);
    if (C > 1) cluster.barrier_wait();
    if (kW > 1 && lane == 0) {
        first->acc[rank_in * kW + warp] = acc;
        first->ahead[rank_in * kW + warp] = ahead;
    }
    if (kW > 1 && acc.s < kNearOne) {  // (only then the row's may be)
        int32_t lead;
        const float others = soft_others(st.acc, acc.m, p.c, lead);
        if (lane == 0) {
            first->others[rank_in * kW + warp] = others;
            first->lead[rank_in * kW + warp] = lead;
        }
    }
    const int32_t slots = int32_t(slot_at - &sh.slot_max[warp][0][lane]) / 32;
    LpShare r{rowp, shift, v_start, v1, stride, per_slot, slots, p.n_top, 0.0f};
    if constexpr (kTop) {
        // the threshold: the n_top-th largest of the groups' maxima
        constexpr int kG = kW == 1 ? 32 : kGroups;
        const int threads = C * kNT / kG;  // of one group: 1 to 32 neighbours
        float most_top = top;
        for (int o = 1; o < threads; o <<= 1) most_top = fmaxf(most_top, __shfl_xor_sync(0xffffffffu, most_top, o));
        if ((lane & (threads - 1)) == 0) {
            const uint32_t k = loom_order_key(most_top);
            const int at = (rank_in * kNT + tid) / threads;
            if (C > 1)
                for (int b = 0; b < C; ++b) cluster.map_shared_rank(&sh, b)->group[at] = k;
            else
                sh.group[at] = k;
        }
        if (C > 1) cluster.sync();
        else block_sync<kW>();
        uint32_t x_key = 0;
        if (p.n_top <= 8) {
            // every warp by itself: the largest, n_top times
            uint32_t k0 = sh.group[lane], k1 = kG > 32 ? sh.group[lane + 32] : 0u;
            for (int i = 0; i < p.n_top; ++i) {
                const uint32_t k = k0 > k1 ? k0 : k1;
                x_key = __reduce_max_sync(0xffffffffu, k);
                if (lane == __ffs(__ballot_sync(0xffffffffu, k == x_key)) - 1) {
                    if (k0 == x_key) k0 = 0;
                    else k1 = 0;
                }
            }
        } else {
            constexpr int kPerKey = kNT / kG;  // threads that count the larger ones of one maximum together
            const int i = tid / kPerKey;
            const uint32_t mine = sh.group[i];
            int larger = 0;
#pragma unroll 2
            for (int j = tid % kPerKey * 4; j < kG; j += kPerKey * 4) {
                const uint4 o = *reinterpret_cast<const uint4*>(&sh.group[j]);
                larger += (o.x > mine || (o.x == mine && j < i)) + (o.y > mine || (o.y == mine && j + 1 < i)) +
                          (o.z > mine || (o.z == mine && j + 2 < i)) + (o.w > mine || (o.w == mine && j + 3 < i));
            }
#pragma unroll
            for (int o = 1; o < kPerKey; o <<= 1) larger += __shfl_xor_sync(0xffffffffu, larger, o);
            if (larger == p.n_top - 1) sh.x_key = mine;
            block_sync<kW>();
            x_key = sh.x_key;
        }
        r.X = order_key_to_float(x_key);
        // the elements that reach it, to the first block
        const int most = LpShared<kW, kTop>::kMaxCand / C;
        uint64_t* to = first->cand + rank_in * most;
        auto add = [&](const float(&x)[4], const int32_t(&id)[4]) {
            uint32_t b[4];
            int n = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                b[k] = __ballot_sync(0xffffffffu, x[k] >= r.X);
                n += __popc(b[k]);
            }
            if (n == 0) return;
            int at = 0;
            if (lane == 0) at = atomicAdd(&sh.n_cand, n);
            at = __shfl_sync(0xffffffffu, at, 0);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int here = at + __popc(b[k] & ((1u << lane) - 1u));
                if (x[k] >= r.X && here < most) to[here] = loom_rank_key(x[k], id[k]);
                at += __popc(b[k]);
            }
        };
        // (a threshold of -inf lets everything through: to the lists at once, in every block alike)
        const bool all = r.X == neg_inf();
        if (all && tid == 0) sh.overflow = 1;
        uint32_t mine = 0;  // this thread's slots whose maximum does
#pragma unroll 4
        for (int32_t s = 0; s < slots && !all; ++s) mine |= uint32_t(sh.slot_max[warp][s][lane] >= r.X) << s;
        const bool own = kW == 1 && p.n_top > 8 && p.width <= kOwnSlots;
        if (own) {
            // most lanes have some (n_top of 32): each looks through its own
            for (; mine; mine &= mine - 1) {
                int32_t v = v_start + lane + (__ffs(mine) - 1) * per_slot * stride;
                for (int i = 0; i < per_slot; ++i, v += stride) {
                    uint4 w[kU];
#pragma unroll
                    for (int u = 0; u < kU; ++u)
                        if (v + u * kNT < v1) w[u] = ldg_stream_v4(vec + int64_t(v + u * kNT) * 16);
#pragma unroll
                    for (int u = 0; u < kU; ++u) {
                        if (v + u * kNT >= v1 || !(vec_max<kDtype>(w[u]) >= r.X)) continue;
                        Vec16<kDtype> e;
                        e.unpack(w[u]);
#pragma unroll
                        for (int q = 0; q < kPer; ++q) {
                            if (e.x[q] >= r.X) {
                                const int at = atomicAdd(&sh.n_cand, 1);
                                if (at < most) to[at] = loom_rank_key(e.x[q], (v + u * kNT) * kPer - shift + q);
                            }
                        }
                    }
                }
            }
            __syncwarp();
        } else {
            for (;;) {  // one slot of every lane that has one
                const uint32_t hits = __ballot_sync(0xffffffffu, mine != 0);
                if (hits == 0) break;
                const int32_t s = mine ? __ffs(mine) - 1 : 0;
                mine &= mine - 1;
                visit<kDtype, kU, kNT>(r, hits, s, add);
            }
        }
        if (const int32_t id = edge_id(); !all && id >= 0 && sh.edge[lane] >= r.X) {
            const int at = atomicAdd(&sh.n_cand, 1);
            if (at < most) to[at] = loom_rank_key(sh.edge[lane], id);
        }
        block_sync<kW>();
        if (tid == 0) {
            const int n = sh.n_cand;
            first->part_cand[rank_in] = n < most ? n : most;
            if (n > most)
                for (int b = 0; b < C; ++b) (C > 1 ? cluster.map_shared_rank(&sh, b) : &sh)->overflow = 1;
        }
    }
    if (C > 1) cluster.sync();
    else block_sync<kW>();

    uint64_t key = 0;
    bool listed = false;
    if constexpr (kTop) {
        listed = sh.overflow != 0;
        if (listed) {  // too many to hand on: each warp sorts its own, then lists by halves, warps and blocks
            key = list_slots<kDtype, kU, kW>(r, &sh);
            if (warp == 0) {
                const int32_t id = edge_id();
                key = merge_lists(key, sort_desc(id >= 0 && sh.edge[lane] >= r.X ? loom_rank_key(sh.edge[lane], id) : 0ull));
            }
            for (int h = kW / 2; h > 0; h >>= 1) {
                if (warp >= h && warp < 2 * h) sh.list[warp][lane] = key;
                block_sync<kW>();
                if (warp < h) key = merge_lists(key, sh.list[warp + h][lane]);
            }
            if (C > 1) {
                if (warp == 0) first->part_list[rank_in][lane] = key;
                cluster.sync();
                if (warp == 0 && rank_in == 0)
                    for (int b = 1; b < C; ++b) key = merge_lists(key, sh.part_list[b][lane]);
            }
        }
    }
    // (nothing of the other blocks' shared memory is read from here on)
    constexpr int kLast = kTop && kW > 1 ? 1 : 0;  // the warp that finishes the row's sums; the first, the alternatives
    if (rank_in != 0 || warp > kLast) return;
    if (kTop && warp == 0 && !listed) {
        // Each candidate's place is the number of larger ones. (They come in a part for each block: candidate i is in the
        // part in whose counts' running sum it falls.)
        const int most = LpShared<kW, kTop>::kMaxCand / C;
        int end = lane < C ? sh.part_cand[lane] : 0;
#pragma unroll
        for (int o = 1; o < LpShared<kW, kTop>::kBlocks; o <<= 1) {
            const int below = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += below;
        }
        const int n = __shfl_sync(0xffffffffu, end, C - 1);
        for (int i0 = 0; i0 < n; i0 += 32) {
            const int i = i0 + lane;
            int part = 0, start = 0;
#pragma unroll
            for (int b = 0; b + 1 < LpShared<kW, kTop>::kBlocks; ++b) {
                const int e = __shfl_sync(0xffffffffu, end, b);
                if (b + 1 < C && i >= e) {
                    part = b + 1;
                    start = e;
                }
            }
            if (i < n) sh.sorting[i] = sh.cand[part * most + i - start];
        }
        if (lane < 8) sh.sorting[n + lane] = 0;  // (below every key)
        sh.list[0][lane] = 0;
        __syncwarp();
        for (int i = lane; i < n; i += 32) {
            const uint64_t mine = sh.sorting[i];
            int larger = 0;
            for (int j = 0; j < n; j += 8) {
#pragma unroll
                for (int q = 0; q < 8; ++q) larger += sh.sorting[j + q] > mine;
            }
            if (larger < p.n_top) sh.list[0][larger] = mine;
        }
        __syncwarp();
        key = sh.list[0][lane];
    }
    // x / T by the reciprocal in two parts; where the product with the first is infinite already, that is it (with the second it
    // may be of the other sign, or NaN)
    auto over_t = [&](float x) {
        const float y = __fmul_rn(x, p.inv_t);
        return fabsf(y) <= FLT_MAX ? __fmaf_rn(x, p.inv_t, __fmul_rn(x, p.inv_t_lo)) : y;
    };
    float m = acc.m, lns = 0.0f;
    if (warp == kLast) {
        if constexpr (kW > 1) {
            acc = soft_init();
            ahead = 0;
            for (int w = lane; w < C * kW; w += 32) {  // (at most two to a lane)
                const SoftAcc other = sh.acc[w];
                const float M = fmaxf(acc.m, other.m);
                const SoftAcc x = soft_move(acc, M, p.c), y = soft_move(other, M, p.c);
                acc = {M, x.s + y.s, x.a + y.a};
                ahead += sh.ahead[w];
            }
            acc = soft_reduce(acc, 32, p.c);
            ahead = __reduce_add_sync(0xffffffffu, ahead);
        }
        m = acc.m;
        lns = logf(acc.s);  // -inf for an empty row, NaN where a logit was NaN or +inf
        if (acc.s > 0.0f && acc.s < kNearOne) {
            // One id has nearly all of the probability, 1 / S, and ln S is a small number that the 1 in S leaves few digits
            // of: the sum again without it, from the parts that do not hold it and the elements of the lane that does
            // (two round trips to L2 more: [20000, 300] bf16 with 20 alternatives, such in every fifth row, 40.0 -> 44.6 us).
            int32_t lead = 0, at = 0;
            float rest;
            if constexpr (kW > 1) {
                at = 64;
                rest = 0.0f;
                for (int w = lane; w < C * kW; w += 32) {
                    const SoftAcc other = sh.acc[w];
                    if (other.m == m && other.s > 0.0f) {
                        at = w;
                        rest += sh.others[w];
                        lead = sh.lead[w];
                    } else {
                        rest += soft_move(other, m, p.c).s;
                    }
                }
                for (int o = 16; o > 0; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
                const int32_t all = __reduce_min_sync(0xffffffffu, at);
                lead = __shfl_sync(0xffffffffu, lead, all % 32);
                at = all;
            } else {
                rest = soft_others(st.acc, m, p.c, lead);
            }
            const int32_t from = v0 + (at / kW) * kU * kNT + (at % kW) * 32 + lead;
            rest += sum_without_max<kDtype, kU, kNT>(vec, from, v1, stride, m, p.c);
            if (const float x = at == 0 ? sh.edge[lead] : m; x != m)
                rest += ex2(fmaxf(__fmul_rn(__fsub_rn(x, m), p.c), kMinExp2));
            lns = log1pf(rest);
            acc.s = 1.0f + rest;
        }
        const bool empty = acc.s == 0.0f;
        if (lane == 0) {
            if (kLast > 0) {
                sh.m = m;
                sh.lns = lns;
            }
            if (p.out_lse) p.out_lse[row] = empty ? neg_inf() : over_t(m) + lns;
            if (p.out_entropy) p.out_entropy[row] = empty ? quiet_nan() : lns - kLn2 * __fdiv_rn(acc.a, acc.s);
            if (p.out_logp) {
                float lp = over_t(__fsub_rn(xt, m)) - lns;
                if (empty || (!has && t >= 0)) lp = quiet_nan();
                p.out_logp[row] = t < 0 ? 0.0f : lp;
            }
            if (p.out_rank) p.out_rank[row] = has && xt == xt ? ahead : -1;
        }
    }
    if constexpr (kTop) {
        if constexpr (kLast > 0) {
            named_barrier(1, 64);
            if (warp != 0) return;
            m = sh.m;
            lns = sh.lns;
        }
        if (lane < p.n_top) {
            if (p.out_top_ids) p.out_top_ids[row * p.n_top + lane] = key ? rank_key_id(key) : -1;
            if (p.out_top_logp)
                p.out_top_logp[row * p.n_top + lane] =
                    lns == neg_inf() || !key ? quiet_nan() : over_t(__fsub_rn(rank_key_value(key), m)) - lns;
        }
    }
}

// Blocks per row: doubled, up to 8 (a portable cluster), while there are fewer than two a SM and more than one step of 16
// elements a thread in each one's share. More blocks read faster, but each has its end to go through: [256, 262144] bf16
// 43.6 us with two blocks a row, 48.1 with four, [77, 51865] bf16 12.4 and 16.2.
// A warp to a row, where its row is short beside the number of rows: those up to 1024 wide for a row or more to an SM
// ([2000, 800] f32 9.2 us, four warps to a row 17.0), to 2048 for four ([700, 2048] bf16 9.9 and 9.2, [1000, 2048] 10.1
// and 11.4), to 8192 for fourteen ([1300, 8000] bf16 25.3 and 19.1, [8000, 8000] 66.1 and 92.6); very short rows always.
// Four warps to a row, up to 8192 wide, for more rows than SMs ([200, 8000] bf16 8.0 us, by clusters 11.2), and any with more
// than four to an SM; with fewer, long rows go by clusters ([590, 32000] f32 21.5 us, four warps 23.4).
constexpr int32_t kNarrow = 8192, kShort = 512;
int lp_cluster(int64_t rows, int64_t n_vocab, int sms) {
    int c = 1;
    while (c < kMaxCluster && rows * c < 2 * int64_t(sms) && n_vocab > int64_t(c) * 16 * kLpWarps * 32) c *= 2;
    return c;
}

template <int kDtype, bool kTop, int kW, int kU>
cudaError_t launch_lp(const LpDev& p, int64_t rows, int C, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(kW == 1 ? (rows + 3) / 4 : rows * C));
    cfg.blockDim = dim3(kW == 1 ? 128 : kW * 32);
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = unsigned(C);
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<kDtype, kTop, kW, kU>, p);
}

template <int kDtype, bool kTop>
cudaError_t launch_lp_any(const LpDev& p, int64_t rows, int sms, cudaStream_t s) {
    const int64_t per_sm = p.width <= 1024 ? 1 : p.width <= 2048 ? 4 : 14;
    if (p.width <= kShort || (p.width <= kNarrow && rows >= per_sm * sms)) {
        constexpr int kStep = 2 * 32 * (kDtype == LOOM_SELECT_BF16 ? 8 : 4);  // a warp's step, kU = 2
        if (p.width <= 2 * kStep) return launch_lp<kDtype, kTop, 1, 2>(p, rows, 1, s);
        return launch_lp<kDtype, kTop, 1, 4>(p, rows, 1, s);
    }
    if (rows > (p.width <= kNarrow ? 1 : 4) * int64_t(sms)) return launch_lp<kDtype, kTop, kLpRowWarps, 4>(p, rows, 1, s);
    const int C = lp_cluster(rows, p.width, sms);
    constexpr int64_t kWide = int64_t(8) * kLpWarps * 32 * (kDtype == LOOM_SELECT_BF16 ? 8 : 4);  // a block's step, kU = 8
    if (rows * C <= sms && p.width >= 2 * C * kWide) return launch_lp<kDtype, kTop, kLpWarps, 8>(p, rows, C, s);
    return launch_lp<kDtype, kTop, kLpWarps, 4>(p, rows, C, s);
}

// ---- the gradient ----
//
// L = sum_r g_r log p_r(t_r) + h_r H_r. With l_j = y_j - lse and p_j = e^(l_j):
//   dL/dx_j = (1/T) [ g (delta_jt - p_j) - h p_j (l_j + H) ]   (dH/dy_j = -p_j (l_j + H)).
// Elementwise once lse and H are there (the forward pass returns them), but for an id with p near 1: lse is an f32, so
// log p is off by half a unit of lse's last place, and 1 - p by as much in absolute terms, of a small number that is the
// row's largest entry. A row's entries add up to zero, and the others' are off by that only relative to themselves: such
// an id's entry is minus the sum of the others. A row therefore belongs to one warp, block or cluster, which joins
// its threads' sums at the end. Bound: HBM ([1024, 151936] f32 in 192 us, 6.5 TB/s).
struct LpGradDev {
    const unsigned char* base;
    int64_t rows, width, row_stride;
    const int32_t* ids;
    double T;
    float inv_t, c;  // 1 / T, log2(e) / T
    const float* lse;
    const float* entropy;
    const float* g_logp;
    const float* g_entropy;
    unsigned char* out;
    int64_t out_stride;
    float likely;       // a likely id's x - lse T is above this
    float low_entropy;  // a row with one has less than this
    bool in_place;
};

template <int kDtype>
__device__ __forceinline__ void store_elem(void* base, int64_t i, float v) {
    if constexpr (kDtype == LOOM_SELECT_BF16) reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<float*>(base)[i] = v;
}

// (plain loads: the gradient may be written over the logits)
template <int kDtype>
__device__ __forceinline__ float plain_elem(const void* base, int64_t i) {
    if constexpr (kDtype == LOOM_SELECT_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[i]);
    else return reinterpret_cast<const float*>(base)[i];
}

__device__ __forceinline__ uint4 plain_v4(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p)
                 : "memory");
    return r;
}

// An id is likely, its entry taken from the others', where log2 p is above this (p above 0.758, so one id of a row at most:
// below it the entry's own error is at most three times p's).
constexpr float kLikely = -0.4f;
// The others' sum is taken where it agrees with the formula's own value to this much, and 2^-22 of lse, of the weights. (The
// forward call's lse is off by about 1e-6 and its rounding. With an lse of more ids than the row's the entries do not add up
// to zero.)
constexpr float kLseError = 1.52587890625e-5f;  // 2^-16

// What a row's elements share. l / ln 2 = ((x - lse T) log2(e) / T), with lse T in two f32 parts: near the row's
// likely elements the first difference is exact, so l is off by what lse is, and a few units of its own size.
struct LpGradRow {
    float hi, lo_c;  // lse T; the second part's product with c, negated
    float g, h;      // the gradient is p (g + h l / ln 2), plus `at` at t
    float c;         // log2(e) / T
    float at;

    __device__ __forceinline__ float exponent(float x) const {
        // (clamped: p is 0 there, and stays finite times l)
        return max_nan(__fmaf_rn(__fsub_rn(x, hi), c, lo_c), kMinExp2);
    }

    __device__ __forceinline__ float grad(float l, bool is_t) const {
        return __fadd_rn(__fmul_rn(ex2(l), __fmaf_rn(h, l, g)), is_t ? at : 0.0f);
    }

    // Two at a time, without `at`.
    __device__ __forceinline__ uint64_t grad2(uint64_t x, uint64_t hi2, uint64_t lo_c2, uint64_t c2, uint64_t h2,
                                              uint64_t g2) const {
        uint64_t l;
        asm("sub.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(hi2));
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(l) : "l"(x), "l"(c2), "l"(lo_c2));
        float l0, l1;
        unpack2(l, l0, l1);
        l0 = max_nan(l0, kMinExp2);
        l1 = max_nan(l1, kMinExp2);
        const uint64_t e = pack2(ex2(l0), ex2(l1));
        l = pack2(l0, l1);
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(x) : "l"(h2), "l"(l), "l"(g2));
        asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(e));
        return x;
    }
};

// Element q of a 16-byte vector, q not known to the compiler.
template <int kDtype>
__device__ __forceinline__ float pick(uint4 raw, int q) {
    const int word = kDtype == LOOM_SELECT_BF16 ? q >> 1 : q;
    const uint32_t a = word & 1 ? raw.y : raw.x, b = word & 1 ? raw.w : raw.z, w = word & 2 ? b : a;
    if constexpr (kDtype == LOOM_SELECT_BF16) return __uint_as_float(q & 1 ? w & 0xffff0000u : w << 16);
    else return __uint_as_float(w);
}

constexpr int kGradNT = 256;  // threads of a block that holds a row to each warp
constexpr int kGradU = 4;
// Shares of a row. A warp: rows of one step, and up to 4096 wide where there are 32 or more to an SM ([16384, 1025] f32 25.6 us,
// blocks of four warps 40.7; [1000, 4000] f32 14.6 and 8.6). A block of sixteen warps, one step, where there is no more
// than a row to an SM ([148, 8000] f32 3.5 us, eight warps 4.5); else of four, two steps ([8000, 8000] bf16 51.5 us, eight
// warps 54.7). Wider rows: a few by clusters of blocks of sixteen warps, a step each while there are blocks (one of 151936
// f32 4.7 us, eight warps 5.5; of 20000 2.5 and 2.8); many by blocks of eight with three to six steps each
// ([1024, 151936] f32, clusters of 8: 191.5 us, 4: 197.5, 2: 203; bf16, 4: 100.6, 2: 103.3, 8: 103.3; [3000, 32000] f32,
// 2: 119.8, 1: 126.6, 8: 137), and with fewer steps where there are less than three blocks to an SM ([77, 51865] bf16,
// 8: 6.7 us, 4: 7.5, 2: 8.2). With a likely id in every row, whose entries have to be summed, [1024, 151936] f32 takes 204 us
// and bf16 112.
constexpr int64_t kGradNarrow = 4096, kGradFew = 4;

// What a block found in its part of a row.
struct GradPart {
    float sum;      // of the entries, the likely id's left out
    float direct;   // its entry by the formula
    int32_t id, n;  // the likely id; how many there were
};

template <int kWarps>
struct GradShared {
    float direct;
    int32_t id;
    float warp_sum[kWarps];
    GradPart part[kWarps > 1 ? kMaxCluster : 1];  // of the cluster's blocks, in its first
};

// A row to kWarps warps in each block of a cluster (kWarps == 1: to a warp, eight rows to a block), kGradU vectors a thread
// and step. Rows of logits and of the gradient that start at the same place within 16 bytes go by vectors, the elements of
// those that the row only partly fills apart; others element by element.
template <int kDtype, int kWarps>
__global__ void __launch_bounds__(kWarps == 1 ? kGradNT : kWarps * 32, kWarps == 4 ? 10 : kWarps == 16 ? 2 : 5)
    token_logprobs_grad_kernel(const LpGradDev p) {
    constexpr int kEsz = kDtype == LOOM_SELECT_BF16 ? 2 : 4;
    constexpr int kPer = 16 / kEsz;
    constexpr int kNT = kWarps * 32;
    constexpr int kRows = kWarps == 1 ? kGradNT / 32 : 1;
    __shared__ GradShared<kWarps> sh_of_row[kRows];
    GradShared<kWarps>& sh = sh_of_row[kWarps == 1 ? threadIdx.x / 32 : 0];
    const cg::cluster_group cluster = cg::this_cluster();
    const int C = kWarps == 1 ? 1 : int(cluster.num_blocks()), rank_in = kWarps == 1 ? 0 : int(cluster.block_rank());
    const int64_t row = kWarps == 1 ? int64_t(blockIdx.x) * kRows + threadIdx.x / 32 : blockIdx.x / unsigned(C);
    const int32_t thread = threadIdx.x % kNT;
    if (kWarps == 1 && row >= p.rows) return;
    const unsigned char* in = p.base + row * p.row_stride * kEsz;
    unsigned char* out = p.out + row * p.out_stride * kEsz;
    const int32_t width = int32_t(p.width), shift = int32_t((reinterpret_cast<uintptr_t>(in) & 15) / kEsz);
    const bool vectors = shift == int32_t((reinterpret_cast<uintptr_t>(out) & 15) / kEsz);

    const int32_t t = p.ids ? p.ids[row] : -1;
    const float g_any = p.g_logp ? p.g_logp[row] : 0.0f;
    const float h = p.g_entropy ? p.g_entropy[row] : 0.0f;
    const float ent = p.g_entropy ? p.entropy[row] : 0.0f;
    const float lse = p.lse[row];
    const float g = t >= 0 ? g_any : 0.0f;
    // vectors [v_first, v_end) are inside the row
    const int32_t v_first = shift ? 1 : 0, v_end = max((shift + width) / kPer, v_first);
    const unsigned char* vin = in - shift * kEsz;
    unsigned char* vout = out - shift * kEsz;
    // the others' elements: the first's by threads 0 .. kPer - 1, the last's by the next kPer
    auto edge = [&] {
        int32_t id = -1;
        if (thread < kPer && v_first > 0) id = thread - shift;
        if (thread >= kPer && thread < 2 * kPer && v_end * kPer < shift + width) id = v_end * kPer - shift + thread - kPer;
        return rank_in == 0 && id < width ? id : -1;
    };
    if (g == 0.0f && h == 0.0f) {
        if (!vectors) {
            for (int32_t id = rank_in * kNT + thread; id < width; id += C * kNT) store_elem<kDtype>(out, id, 0.0f);
        } else {
            if (const int32_t id = edge(); id >= 0) store_elem<kDtype>(out, id, 0.0f);
            for (int32_t v = v_first + rank_in * kNT + thread; v < v_end; v += C * kNT)
                *reinterpret_cast<uint4*>(vout + int64_t(v) * 16) = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    // The vectors of the next step are requested as those of this one are done with.
    int32_t v = vectors ? v_first + rank_in * kGradU * kNT + thread : v_end;
    uint4 raw[kGradU];
#pragma unroll
    for (int u = 0; u < kGradU; ++u)
        if (v + u * kNT < v_end) raw[u] = plain_v4(vin + int64_t(v + u * kNT) * 16);
    const int32_t edge_id = vectors ? edge() : -1;
    const float edge_x = edge_id >= 0 ? plain_elem<kDtype>(in, edge_id) : 0.0f;
    // (its own logit may be gone when the gradient is written over it)
    const float xt = h == 0.0f && !p.in_place && t >= 0 && t < width ? plain_elem<kDtype>(in, t) : 0.0f;
    LpGradRow r;
    const double lt = double(lse) * p.T;
    r.hi = __double2float_rn(lt);
    r.c = p.c;
    r.lo_c = -__fmul_rn(__double2float_rn(lt - double(r.hi)), p.c);
    r.at = __fmul_rn(g, p.inv_t);
    const float hs = __fmul_rn(h, p.inv_t);
    r.g = h != 0.0f ? -__fmaf_rn(hs, ent, r.at) : -r.at;
    r.h = -__fmul_rn(hs, kLn2);
    // an id past the vocabulary, an empty row, a row with NaN or +inf: NaN throughout
    if (!(fabsf(lse) <= FLT_MAX) || (t >= width && g != 0.0f)) r.g = quiet_nan();
    const uint64_t hi2 = pack2(r.hi, r.hi), lo_c2 = pack2(r.lo_c, r.lo_c), c2 = pack2(r.c, r.c), h2 = pack2(r.h, r.h),
                   g2 = pack2(r.g, r.g);
    // Whether the row may have a likely id whose entry matters: any with an entropy term, else the given token.
    const bool sums = h != 0.0f ? ent < p.low_entropy : t < width && (p.in_place || __fsub_rn(xt, r.hi) > p.likely);
    if (C > 1 && sums) cluster.barrier_arrive();  // (waited for before the first remote store: all blocks have begun)
    uint64_t sum2 = 0;
    float sum = 0.0f;
    bool found = false;
    // one element apart from the pairs
    auto element = [&](float x, int32_t id) {
        const float d = r.grad(r.exponent(x), id == t);
        if (sums && __fsub_rn(x, r.hi) > p.likely) {
            if (found) sum = quiet_nan();  // (two: an lse of other logits; nothing is made of the sum)
            found = true;
            sh.direct = d;
            sh.id = id;
        } else {
            sum += d;
        }
        store_elem<kDtype>(out, id, d);
    };
    if (!vectors) {
#pragma unroll 1
        for (int32_t id = rank_in * kNT + thread; id < width; id += C * kNT) element(plain_elem<kDtype>(in, id), id);
    } else {
        if (edge_id >= 0) element(edge_x, edge_id);
#pragma unroll 1
        for (; v < v_end; v += C * kGradU * kNT) {
#pragma unroll
            for (int u = 0; u < kGradU; ++u) {
                if (v + u * kNT >= v_end) break;
                const int32_t first = (v + u * kNT) * kPer - shift;
                unsigned char* to = vout + int64_t(v + u * kNT) * 16;
                const int32_t next = v + u * kNT + C * kGradU * kNT;
                if (uint32_t(t) - uint32_t(first) < uint32_t(kPer) ||
                    (sums && __fsub_rn(vec_max<kDtype>(raw[u]), r.hi) > p.likely)) {
#pragma unroll 1
                    for (int q = 0; q < kPer; ++q) element(pick<kDtype>(raw[u], q), first + q);
                    if (next < v_end) raw[u] = plain_v4(vin + int64_t(next) * 16);
                    continue;
                }
                const Pairs<kDtype> x(raw[u]);
                uint32_t w[4];
#pragma unroll
                for (int q = 0; q < kPer / 2; ++q) {
                    const uint64_t d2 = r.grad2(x.v[q], hi2, lo_c2, c2, h2, g2);
                    add2(sum2, d2);
                    float d0, d1;
                    unpack2(d2, d0, d1);
                    if constexpr (kDtype == LOOM_SELECT_BF16) {
                        const __nv_bfloat162 pr = __floats2bfloat162_rn(d0, d1);
                        w[q] = *reinterpret_cast<const uint32_t*>(&pr);
                    } else {
                        w[2 * q] = __float_as_uint(d0), w[2 * q + 1] = __float_as_uint(d1);
                    }
                }
                if (next < v_end) raw[u] = plain_v4(vin + int64_t(next) * 16);
                *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
    if (!sums) return;  // (the whole row's threads)
    float s0, s1;
    unpack2(sum2, s0, s1);
    sum += s0 + s1;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    GradPart all;
    all.sum = sum;
    if constexpr (kWarps == 1) {
        all.n = __popc(__ballot_sync(0xffffffffu, found));
        __syncwarp();
    } else {
        if (threadIdx.x % 32 == 0) sh.warp_sum[threadIdx.x / 32] = sum;
        all.n = __syncthreads_count(found);
    }
    all.direct = sh.direct, all.id = sh.id;
    if constexpr (kWarps > 1) {
        if (thread == 0) {
            all.sum = 0.0f;
            for (int w = 0; w < kWarps; ++w) all.sum += sh.warp_sum[w];
        }
        if (C > 1) {
            cluster.barrier_wait();
            if (thread == 0) *cluster.map_shared_rank(&sh.part[rank_in], 0) = all;
            cluster.sync();
            if (rank_in != 0) return;  // (nobody reads this block's shared memory)
            if (thread == 0) {
                all = sh.part[0];
                for (int b = 1; b < C; ++b) {
                    const GradPart o = sh.part[b];
                    all.sum += o.sum;
                    if (o.n) all.direct = o.direct, all.id = o.id;
                    all.n += o.n;
                }
            }
        }
    }
    if (thread != 0 || all.n != 1) return;
    const float g_abs = p.g_logp && t >= 0 ? fabsf(p.g_logp[row]) : 0.0f, h_abs = p.g_entropy ? fabsf(p.g_entropy[row]) : 0.0f;
    const float weight = g_abs + (h_abs != 0.0f ? h_abs * (4.0f + 2.0f * p.entropy[row]) : 0.0f);
    const float off = weight * p.inv_t * (kLseError + 2.0f * FLT_EPSILON * fabsf(p.lse[row]));
    if (fabsf(-all.sum - all.direct) <= off) store_elem<kDtype>(out, all.id, -all.sum);
}

template <int kDtype, int kWarps>
cudaError_t launch_grad(const LpGradDev& p, int C, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(kWarps == 1 ? (p.rows + kGradNT / 32 - 1) / (kGradNT / 32) : p.rows * C));
    cfg.blockDim = dim3(kWarps == 1 ? kGradNT : kWarps * 32);
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = unsigned(C);
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, token_logprobs_grad_kernel<kDtype, kWarps>, p);
}

template <int kDtype>
cudaError_t launch_grad_any(const LpGradDev& p, int sms, cudaStream_t s) {
    constexpr int kPer = kDtype == LOOM_SELECT_BF16 ? 8 : 4;
    const int64_t nv = (p.width + kPer - 2) / kPer + 1;  // (a row may start inside a vector)
    auto steps = [&](int warps) { return (nv + warps * 32 * kGradU - 1) / (warps * 32 * kGradU); };
    if (steps(1) == 1 || (p.width <= kGradNarrow && p.rows >= 32 * int64_t(sms))) return launch_grad<kDtype, 1>(p, 1, s);
    if (steps(16) == 1 && p.rows <= sms) return launch_grad<kDtype, 16>(p, 1, s);
    if (steps(4) <= 2) return launch_grad<kDtype, 4>(p, 1, s);
    int C = 1;
    if (p.rows <= kGradFew) {
        while (C < kMaxCluster && steps(16) > C) C *= 2;
        return launch_grad<kDtype, 16>(p, C, s);
    }
    while (C < kMaxCluster && (steps(8) >= 6 * C || (steps(8) > C && p.rows * C < 3 * int64_t(sms)))) C *= 2;
    return launch_grad<kDtype, 8>(p, C, s);
}

bool dtype_ok(int dtype) { return dtype == LOOM_SELECT_F32 || dtype == LOOM_SELECT_BF16; }
size_t esz_of(int dtype) { return dtype == LOOM_SELECT_BF16 ? 2 : 4; }
bool misaligned(const void* p, size_t a) { return p && reinterpret_cast<uintptr_t>(p) % a != 0; }

// A normal number: 1 / T and log2(e) / T are finite then. (Where they are subnormal, for T above 8.5e37, they are off by 2e-7 of
// themselves and x / T is below 4.)
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
    p.rows = rows;
    p.c = float(1.4426950408889634 / double(temperature));
    p.inv_t = float(1.0 / double(temperature));
    p.inv_t_lo = float(1.0 / double(temperature) - double(p.inv_t));
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
    const auto s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (dtype == LOOM_SELECT_BF16)
        e = n_top ? launch_lp_any<LOOM_SELECT_BF16, true>(p, rows, sms, s)
                  : launch_lp_any<LOOM_SELECT_BF16, false>(p, rows, sms, s);
    else
        e = n_top ? launch_lp_any<LOOM_SELECT_F32, true>(p, rows, sms, s)
                  : launch_lp_any<LOOM_SELECT_F32, false>(p, rows, sms, s);
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
    p.rows = rows;
    p.width = n_vocab;
    p.row_stride = row_stride;
    p.ids = ids;
    p.T = double(temperature);
    p.inv_t = float(1.0 / double(temperature));
    p.c = float(1.4426950408889634 / double(temperature));
    p.lse = lse;
    p.entropy = entropy;
    p.g_logp = grad_logp;
    p.g_entropy = grad_entropy;
    p.out = static_cast<unsigned char*>(out_grad);
    p.out_stride = grad_stride;
    p.likely = float(kLikely * 0.6931471805599453 * p.T);
    p.low_entropy = float(0.57 + 0.25 * std::log(double(n_vocab)));  // (at p = 3/4, the rest evenly spread: 0.563 + ln(V - 1) / 4)
    p.in_place = logits == out_grad;
    const auto s = static_cast<cudaStream_t>(stream);
    int st = LOOM_SELECT_OK;
    const int sms = device_sm_count(&st);
    if (st != LOOM_SELECT_OK) return st;
    const cudaError_t e = dtype == LOOM_SELECT_BF16 ? launch_grad_any<LOOM_SELECT_BF16>(p, sms, s)
                                                    : launch_grad_any<LOOM_SELECT_F32>(p, sms, s);
    return e == cudaSuccess ? LOOM_SELECT_OK : LOOM_SELECT_ECUDA;
}

}  // extern "C"
