// select_quant.cu -- rows to 8-bit integers with a scale per row: behind the final RMS norm, or as they are.
//
// rms_norm_i8, per row, with D = dim:
//   h = x + r          one rounding to the rows' type (stored to out_sum where asked for; h = x without r)
//   inv = 1 / sqrt(sum h^2 / D + eps)      in 64 bits, rounded once to f32
//   y = (h * inv) * w                      two f32 roundings
//   a = max |y|,  scale = a / 127,  q = rint(y * ((1 / a) * 127))      each step one f32 rounding, |q| <= 127
// quantize_rows_i8 takes y = x. The sum of squares is held in 64 bits, where the order of the summation shows only
// at 2^-53: the one rounding of inv to f32 comes out the same for any order, and q as the plain definition gives it
// whatever the launch shape, but for about one row in 10^8.
// Bound: HBM (rows read once: a thread keeps its elements in registers between the passes). [16384, 4096] f32 with the
// residual takes 127.5 us (6.8 TB/s), [16384, 2048] bf16 38.5 us (6.1 TB/s), one row 2.8 us.
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cuda_runtime.h>

#include "loom_select.h"
#include "select_device.cuh"
#include "select_internal.h"
#include "select_rows.cuh"

namespace loom_select {
namespace {

// A row whose largest magnitude is below this counts as zero (its reciprocal would leave f32's range).
constexpr float kTinyRow = 7.888609052210118e-31f;  // 2^-100
constexpr int kMaxDim = 32768;

struct QuantDev {
    const unsigned char* x;
    const unsigned char* residual;
    const unsigned char* weight;
    unsigned char* sum;
    int8_t* q;
    float* scale;
    int64_t rows;
    int64_t x_stride, residual_stride, sum_stride;
    int32_t dim;
    double eps;
};

__device__ __forceinline__ float nan_max(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// The 16-byte vectors around kWords 32-bit words that begin at a multiple of 2.
template <int kWords>
struct Around {
    static constexpr int kVecs = (kWords + 3) / 4 + 1;
    uint32_t w[4 * kVecs];
    __device__ __forceinline__ void load(const unsigned char* at, bool there) {
        const uint4* v = reinterpret_cast<const uint4*>(at - (reinterpret_cast<uintptr_t>(at) & 15));
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            uint4 r = make_uint4(0, 0, 0, 0);
            if (there) r = v[i];
            w[4 * i] = r.x, w[4 * i + 1] = r.y, w[4 * i + 2] = r.z, w[4 * i + 3] = r.w;
        }
    }
    // The words themselves. The shift is the same for a whole row's runs, so the branches are uniform.
    __device__ __forceinline__ void get(const unsigned char* at, uint32_t (&out)[kWords]) const {
        const uint32_t s = uint32_t(reinterpret_cast<uintptr_t>(at) & 15), bits = (s & 2) * 8;
#pragma unroll
        for (int skip = 0; skip < 4; ++skip) {
            if (s >> 2 == skip) {
#pragma unroll
                for (int q = 0; q < kWords; ++q) out[q] = __funnelshift_r(w[q + skip], w[q + skip + 1], bits);
            }
        }
    }
};

// kN neighbouring elements of a whole run, as raw words; zeros where there is none. kAligned: the address is a multiple of
// their size (at most 16 bytes). Otherwise the vectors around them lie in the same row (see kBefore); f32 runs of four go
// word by word, which is quicker ([30000, 1037] with the residual 108 us, by vectors 142, as both then stood).
template <int kDtype, int kN, bool kAligned>
struct RunLoad {
    static constexpr int kWords = kN * (kDtype == LOOM_SELECT_BF16 ? 2 : 4) / 4;
    static constexpr bool kByWord = !kAligned && kDtype == LOOM_SELECT_F32 && kN == 4;
    Around<kWords> around;  // (its first words are the run itself where it is not loaded around it)
    const unsigned char* at;
    __device__ __forceinline__ void load(const unsigned char* from, bool there) {
        at = from;
        if constexpr (!kAligned && !kByWord) {
            around.load(at, there);
        } else {
#pragma unroll
            for (int q = 0; q < kWords; ++q) around.w[q] = 0;
            if (!there) return;
            if constexpr (kByWord) {
#pragma unroll
                for (int q = 0; q < kWords; ++q) around.w[q] = reinterpret_cast<const uint32_t*>(at)[q];
            } else if constexpr (kWords == 2) {
                const uint2 r = *reinterpret_cast<const uint2*>(at);
                around.w[0] = r.x, around.w[1] = r.y;
            } else {
#pragma unroll
                for (int q = 0; q < kWords; q += 4) {
                    const uint4 r = *reinterpret_cast<const uint4*>(at + 4 * q);
                    around.w[q] = r.x, around.w[q + 1] = r.y, around.w[q + 2] = r.z, around.w[q + 3] = r.w;
                }
            }
        }
    }
    __device__ __forceinline__ void get(uint32_t (&out)[kWords]) const {
        if constexpr (!kAligned && !kByWord) {
            around.get(at, out);
        } else {
#pragma unroll
            for (int q = 0; q < kWords; ++q) out[q] = around.w[q];
        }
    }
};

template <int kDtype, int kWords, int kN>
__device__ __forceinline__ void words_to_floats(const uint32_t (&w)[kWords], float (&x)[kN]) {
#pragma unroll
    for (int q = 0; q < kWords; ++q) {
        if constexpr (kDtype == LOOM_SELECT_BF16) {
            x[2 * q] = __uint_as_float(w[q] << 16);
            x[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
        } else {
            x[q] = __uint_as_float(w[q]);
        }
    }
}

// The four words of a whole run to any element-aligned address (kAligned: a multiple of 16).
template <bool kAligned>
__device__ __forceinline__ void store_run(unsigned char* at, const uint32_t (&w)[4]) {
    if constexpr (kAligned) {
        *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
    } else if ((reinterpret_cast<uintptr_t>(at) & 2) == 0) {
#pragma unroll
        for (int q = 0; q < 4; ++q) reinterpret_cast<uint32_t*>(at)[q] = w[q];
    } else {  // bf16 between words
        *reinterpret_cast<unsigned short*>(at) = (unsigned short)w[0];
#pragma unroll
        for (int q = 0; q < 3; ++q) *reinterpret_cast<uint32_t*>(at + 2 + 4 * q) = __funnelshift_r(w[q], w[q + 1], 16);
        *reinterpret_cast<unsigned short*>(at + 14) = (unsigned short)(w[3] >> 16);
    }
}

template <int kDtype>
__device__ __forceinline__ float load_one(const unsigned char* base, int32_t i) {
    if constexpr (kDtype == LOOM_SELECT_BF16)
        return __uint_as_float(uint32_t(reinterpret_cast<const unsigned short*>(base)[i]) << 16);
    else
        return reinterpret_cast<const float*>(base)[i];
}

// A thread's kPer elements in the rows' own type, four registers: f32 x 4 or bf16 x 8.
template <int kDtype>
struct Held {
    static constexpr int kPer = kDtype == LOOM_SELECT_BF16 ? 8 : 4;
    uint32_t w[4];
    __device__ __forceinline__ void get(float (&x)[kPer]) const { words_to_floats<kDtype>(w, x); }
    __device__ __forceinline__ void set(const float (&x)[kPer]) {  // rounds to the type
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if constexpr (kDtype == LOOM_SELECT_BF16) {
                const __nv_bfloat162 t = __floats2bfloat162_rn(x[2 * q], x[2 * q + 1]);
                w[q] = *reinterpret_cast<const uint32_t*>(&t);
            } else {
                w[q] = __float_as_uint(x[q]);
            }
        }
    }
};

// kTPR threads hold one row, kVPT runs of kPer neighbouring elements each, kTPR runs apart; a block holds one row, or
// several of those a warp or less holds. All of a thread's loads are in flight together, and its elements stay in
// registers. Runs are laid out by the output: run k covers ids [k kPer - lead, (k + 1) kPer - lead), where out_q's row
// begins `lead` bytes after a multiple of kPer, so that a whole run is one store. kAligned: every row of every tensor
// begins at a vector (lead is 0). Otherwise runs within kBefore elements of the row's start or kAfter of its end are
// left to single elements, at most 30 of them, so that the vectors around the others' elements lie in the row. (With the
// odd elements inside each run's code, the loads of one run waited for the branches of the one before: [8192, 5001]
// bf16 120 us, this way 86, the bytes 44; [100000, 1501] bf16 quantised 137 and 94, the bytes 69.)
constexpr int kBefore = 8, kAfter = 16;
constexpr int kMaxEdge = 32;
//
// Resident threads per SM asked of the compiler: 1024 (64 registers) where it takes registers to keep the loads in flight,
// 1536 (40) for the plain aligned quantiser, whose [151936, 2048] bf16 takes 132.5 us then (1024: 134.7; the bytes at
// the copy rate 142.8); two blocks of 1024 threads where that is the block ([8192, 16384] f32 96.9 us; one: 128).
constexpr int min_blocks(bool norm, bool aligned, int threads) {
    return norm || !aligned ? 1024 / threads : threads == 1024 ? 2 : 1536 / threads;
}

template <int kDtype, int kWDtype, bool kNorm, int kTPR, int kVPT, bool kAligned>
__global__ void __launch_bounds__(kTPR < 64 ? 128 : kTPR, min_blocks(kNorm, kAligned, kTPR < 64 ? 128 : kTPR))
    quant_rows_kernel(const QuantDev p) {
    constexpr int kEsz = kDtype == LOOM_SELECT_BF16 ? 2 : 4;
    constexpr int kPer = 16 / kEsz;
    constexpr int kWarps = kTPR / 32;  // 0: several rows to a warp
    constexpr int kRows = kTPR < 64 ? 128 / kTPR : 1;
    // y in f32 where a thread has few elements; with many, bf16 rows make it again for the output (from the row and
    // the weight in L1)
    constexpr bool kHoldY = kNorm && (kDtype == LOOM_SELECT_F32 || kVPT <= 4);
    __shared__ double part_ss[kWarps > 1 ? kWarps : 1];
    __shared__ float part_max[kWarps > 1 ? kWarps : 1];
    __shared__ float row_inv;
    const int tid = threadIdx.x % kTPR, lane = tid & 31, warp = tid >> 5;
    const int64_t row_or_past = int64_t(blockIdx.x) * kRows + threadIdx.x / kTPR;
    const bool there = kRows == 1 || row_or_past < p.rows;  // (warps stay whole: rows past the last do nothing)
    const int64_t row = there ? row_or_past : 0;
    const int32_t dim = there ? p.dim : 0;
    unsigned char* out = reinterpret_cast<unsigned char*>(p.q + row * p.dim);
    const int32_t lead = kAligned ? 0 : int32_t(reinterpret_cast<uintptr_t>(out) % kPer);
    auto first = [&](int j) { return (j * kTPR + tid) * kPer - lead; };
    auto whole = [&](int j) {
        return kAligned ? first(j) + kPer <= dim : first(j) >= kBefore && first(j) + kAfter <= dim;
    };
    // the single elements: ids [0, edge0) and [edge1, dim)
    constexpr int kEdge = kAligned ? 0 : (kMaxEdge + kTPR - 1) / kTPR;
    int32_t edge0 = 0, edge1 = dim;
    if constexpr (!kAligned) {
        const int32_t k0 = (kBefore + lead + kPer - 1) / kPer, k1 = dim >= kAfter ? (dim - kAfter + lead) / kPer : -1;
        edge0 = k1 < k0 ? dim : k0 * kPer - lead;
        edge1 = k1 < k0 ? dim : (k1 + 1) * kPer - lead;
    }
    auto edge_id = [&](int i) {
        const int32_t e = i * kTPR + tid;
        return e < edge0 ? e : edge1 + (e - edge0);  // (dim or more: none)
    };

    Held<kDtype> h[kVPT];
    float he[kEdge > 0 ? kEdge : 1];
    auto load_row = [&](const unsigned char* base, Held<kDtype>(&to)[kVPT], float(&edge)[kEdge > 0 ? kEdge : 1]) {
        RunLoad<kDtype, kPer, kAligned> run[kVPT];  // (all requested before the first is shifted)
#pragma unroll
        for (int j = 0; j < kVPT; ++j) run[j].load(base + int64_t(first(j)) * kEsz, whole(j));
#pragma unroll
        for (int i = 0; i < kEdge; ++i) edge[i] = edge_id(i) < dim ? load_one<kDtype>(base, edge_id(i)) : 0.0f;
#pragma unroll
        for (int j = 0; j < kVPT; ++j) run[j].get(to[j].w);
    };
    load_row(p.x + row * p.x_stride * kEsz, h, he);
    if (kNorm && p.residual) {
        unsigned char* s = p.sum ? p.sum + row * p.sum_stride * kEsz : nullptr;
        Held<kDtype> add[kVPT];
        float add_e[kEdge > 0 ? kEdge : 1];
        load_row(p.residual + row * p.residual_stride * kEsz, add, add_e);
#pragma unroll
        for (int j = 0; j < kVPT; ++j) {
            float v[kPer], u[kPer];
            h[j].get(v);
            add[j].get(u);
#pragma unroll
            for (int q = 0; q < kPer; ++q) v[q] = __fadd_rn(v[q], u[q]);
            h[j].set(v);
            if (s && whole(j)) store_run<kAligned>(s + int64_t(first(j)) * kEsz, h[j].w);
        }
#pragma unroll
        for (int i = 0; i < kEdge; ++i) {
            he[i] = __fadd_rn(he[i], add_e[i]);
            if constexpr (kDtype == LOOM_SELECT_BF16) he[i] = __bfloat162float(__float2bfloat16_rn(he[i]));
            if (s && edge_id(i) < dim) {
                if constexpr (kDtype == LOOM_SELECT_BF16)
                    reinterpret_cast<__nv_bfloat16*>(s)[edge_id(i)] = __float2bfloat16_rn(he[i]);
                else
                    reinterpret_cast<float*>(s)[edge_id(i)] = he[i];
            }
        }
    }
    float inv = 0.0f;
    if constexpr (kNorm) {
        double ss = 0.0;
#pragma unroll
        for (int j = 0; j < kVPT; ++j) {
            float v[kPer];
            h[j].get(v);
#pragma unroll
            for (int q = 0; q < kPer; ++q) ss = __fma_rn(double(v[q]), double(v[q]), ss);
        }
#pragma unroll
        for (int i = 0; i < kEdge; ++i) ss = __fma_rn(double(he[i]), double(he[i]), ss);
#pragma unroll
        for (int o = (kTPR < 32 ? kTPR : 32) / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        // (64-bit division and square root by one warp: every warp's would take turns at the unit)
        auto inverse = [&](double sum) {
            return __double2float_rn(__drcp_rn(__dsqrt_rn(__ddiv_rn(sum, double(p.dim)) + p.eps)));
        };
        if constexpr (kWarps > 1) {
            if (lane == 0) part_ss[warp] = ss;
            __syncthreads();
            if (warp == 0) {
                ss = part_ss[0];
#pragma unroll
                for (int w = 1; w < kWarps; ++w) ss += part_ss[w];
                inv = inverse(ss);
                if (lane == 0) row_inv = inv;
            }
            __syncthreads();
            inv = row_inv;
        } else {
            inv = inverse(ss);
        }
    }
    auto make = [&](int j, float (&v)[kPer]) {
        h[j].get(v);
        if constexpr (kNorm) {
            constexpr int kWEsz = kWDtype == LOOM_SELECT_BF16 ? 2 : 4;
            RunLoad<kWDtype, kPer, kAligned> run;
            run.load(p.weight + int64_t(first(j)) * kWEsz, whole(j));
            uint32_t raw[kPer * kWEsz / 4];
            run.get(raw);
            float w[kPer];
            words_to_floats<kWDtype>(raw, w);
#pragma unroll
            for (int q = 0; q < kPer; ++q) v[q] = __fmul_rn(__fmul_rn(v[q], inv), w[q]);
        }
    };
#pragma unroll
    for (int i = 0; i < kEdge; ++i)
        if (kNorm && edge_id(i) < dim) he[i] = __fmul_rn(__fmul_rn(he[i], inv), load_one<kWDtype>(p.weight, edge_id(i)));
    float y[kHoldY ? kVPT : 1][kPer];
    float a = 0.0f;
#pragma unroll
    for (int j = 0; j < kVPT; ++j) {
        float v[kPer];
        make(j, v);
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
            a = nan_max(a, fabsf(v[q]));
            if constexpr (kHoldY) y[j][q] = v[q];
        }
    }
#pragma unroll
    for (int i = 0; i < kEdge; ++i) a = nan_max(a, fabsf(he[i]));
#pragma unroll
    for (int o = (kTPR < 32 ? kTPR : 32) / 2; o > 0; o >>= 1) a = nan_max(a, __shfl_xor_sync(0xffffffffu, a, o));
    if constexpr (kWarps > 1) {
        if (lane == 0) part_max[warp] = a;
        __syncthreads();
        a = part_max[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) a = nan_max(a, part_max[w]);
    }
    // a NaN or an infinity anywhere: q 0 and a NaN scale, so that what is made of them is NaN
    const bool fine = a <= FLT_MAX, some = fine && a >= kTinyRow;
    const float inv_scale = some ? __fmul_rn(__frcp_rn(a), 127.0f) : 0.0f;
    if (tid == 0 && there) p.scale[row] = !fine ? __int_as_float(0x7fc00000) : some ? __fdiv_rn(a, 127.0f) : 0.0f;
    // rint by adding 1.5 * 2^23 (to nearest even): the sum's low byte is the two's complement 8-bit integer
    constexpr float kMagic = 12582912.0f;
#pragma unroll
    for (int j = 0; j < kVPT; ++j) {
        float v[kPer];
        if constexpr (kHoldY) {
#pragma unroll
            for (int q = 0; q < kPer; ++q) v[q] = y[j][q];
        } else {
            make(j, v);
        }
        uint32_t w[kPer / 4];
#pragma unroll
        for (int k = 0; k < kPer / 4; ++k) {
            uint32_t b[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) b[q] = __float_as_uint(__fadd_rn(__fmul_rn(v[4 * k + q], inv_scale), kMagic));
            w[k] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
            if (!some) w[k] = 0;  // (a NaN row's products are not numbers)
        }
        if (whole(j)) {
            if constexpr (kPer == 8) *reinterpret_cast<uint2*>(out + first(j)) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint32_t*>(out + first(j)) = w[0];
        }
    }
#pragma unroll
    for (int i = 0; i < kEdge; ++i) {
        const uint32_t b = __float_as_uint(__fadd_rn(__fmul_rn(he[i], inv_scale), kMagic));
        if (edge_id(i) < dim) out[edge_id(i)] = some ? (unsigned char)b : (unsigned char)0;
    }
}

bool multiple_of(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

template <int kDtype, int kWDtype, bool kNorm, int kTPR, int kVPT, bool kAligned>
void launch_rows(const QuantDev& p, cudaStream_t s) {
    constexpr int kRows = kTPR < 64 ? 128 / kTPR : 1;
    quant_rows_kernel<kDtype, kWDtype, kNorm, kTPR, kVPT, kAligned>
        <<<unsigned((p.rows + kRows - 1) / kRows), kTPR * kRows, 0, s>>>(p);
}

// Threads for a row: as few as hold it at four runs each, since they have many loads in flight and little to join;
// more, up to a run each, when the rows do not give every SM 256 threads ([1024, 1025] f32 3.0 us; with 1024 threads
// asked for 4.6).
template <int kDtype, int kWDtype, bool kNorm, bool kAligned>
void launch_any(const QuantDev& p, int sms, cudaStream_t s) {
    constexpr int kPer = kDtype == LOOM_SELECT_BF16 ? 8 : 4;
    const int nv = (p.dim + (kAligned ? 0 : kPer - 1) + kPer - 1) / kPer;
    int tpr = 8;
    while (tpr < 1024 && (nv > tpr * 4 || (tpr < nv && p.rows * tpr < int64_t(sms) * 256))) tpr *= tpr == 8 ? 4 : 2;
    if (tpr == 8) launch_rows<kDtype, kWDtype, kNorm, 8, 4, kAligned>(p, s);
    else if (tpr == 32) launch_rows<kDtype, kWDtype, kNorm, 32, 4, kAligned>(p, s);
    else if (tpr == 64) launch_rows<kDtype, kWDtype, kNorm, 64, 4, kAligned>(p, s);
    else if (tpr == 128) launch_rows<kDtype, kWDtype, kNorm, 128, 4, kAligned>(p, s);
    else if (tpr == 256) launch_rows<kDtype, kWDtype, kNorm, 256, 4, kAligned>(p, s);
    else if (tpr == 512) launch_rows<kDtype, kWDtype, kNorm, 512, 4, kAligned>(p, s);
    else if (nv <= 1024 * 4) launch_rows<kDtype, kWDtype, kNorm, 1024, 4, kAligned>(p, s);
    else launch_rows<kDtype, kWDtype, kNorm, 1024, kAligned ? 8 : 9, kAligned>(p, s);
}

template <int kDtype, int kWDtype, bool kNorm>
cudaError_t launch_quant_t(const QuantDev& p, int sms, cudaStream_t s) {
    constexpr int kPer = kDtype == LOOM_SELECT_BF16 ? 8 : 4;
    const bool aligned = p.dim % kPer == 0 && p.x_stride % kPer == 0 && p.residual_stride % kPer == 0 &&
                         p.sum_stride % kPer == 0 && multiple_of(p.x, 16) && multiple_of(p.residual, 16) &&
                         multiple_of(p.sum, 16) && multiple_of(p.weight, 16) && multiple_of(p.q, kPer);
    if (aligned) launch_any<kDtype, kWDtype, kNorm, true>(p, sms, s);
    else launch_any<kDtype, kWDtype, kNorm, false>(p, sms, s);
    return cudaGetLastError();
}

bool dtype_ok(int dtype) { return dtype == LOOM_SELECT_F32 || dtype == LOOM_SELECT_BF16; }
size_t esz_of(int dtype) { return dtype == LOOM_SELECT_BF16 ? 2 : 4; }
bool misaligned(const void* p, size_t a) { return p && reinterpret_cast<uintptr_t>(p) % a != 0; }

}  // namespace
}  // namespace loom_select

using namespace loom_select;

extern "C" {

LOOM_SELECT_API int loom_rms_norm_i8(const void* x, int dtype, int64_t rows, int64_t dim, int64_t x_stride,
                                     const void* residual, int64_t residual_stride, const void* weight,
                                     int weight_dtype, double eps, int8_t* out_q, float* out_scale, void* out_sum,
                                     int64_t sum_stride, void* stream) {
    if (!dtype_ok(dtype) || !dtype_ok(weight_dtype)) return LOOM_SELECT_EDTYPE;
    if (!x || !weight || !out_q || !out_scale || rows <= 0 || dim <= 0 || x_stride < dim) return LOOM_SELECT_EINVAL;
    if ((residual && residual_stride < dim) || (out_sum && (!residual || sum_stride < dim))) return LOOM_SELECT_EINVAL;
    // in place only element for element
    if (out_sum && ((out_sum == x && sum_stride != x_stride) || (out_sum == residual && sum_stride != residual_stride)))
        return LOOM_SELECT_EINVAL;
    const size_t esz = esz_of(dtype);
    if (misaligned(x, esz) || misaligned(residual, esz) || misaligned(out_sum, esz) ||
        misaligned(weight, esz_of(weight_dtype)) || misaligned(out_scale, 4))
        return LOOM_SELECT_EINVAL;
    if (!(eps > 0.0) || std::isinf(eps)) return LOOM_SELECT_EPARAM;
    if (dim > kMaxDim || rows > INT32_MAX) return LOOM_SELECT_ESHAPE;
    QuantDev p{};
    p.x = static_cast<const unsigned char*>(x);
    p.residual = static_cast<const unsigned char*>(residual);
    p.weight = static_cast<const unsigned char*>(weight);
    p.sum = static_cast<unsigned char*>(out_sum);
    p.q = out_q;
    p.scale = out_scale;
    p.rows = rows;
    p.x_stride = x_stride;
    p.residual_stride = residual_stride;
    p.sum_stride = sum_stride;
    p.dim = int32_t(dim);
    p.eps = eps;
    int st = LOOM_SELECT_OK;
    const int sms = device_sm_count(&st);
    if (st != LOOM_SELECT_OK) return st;
    const auto s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (dtype == LOOM_SELECT_BF16)
        e = weight_dtype == LOOM_SELECT_BF16 ? launch_quant_t<LOOM_SELECT_BF16, LOOM_SELECT_BF16, true>(p, sms, s)
                                             : launch_quant_t<LOOM_SELECT_BF16, LOOM_SELECT_F32, true>(p, sms, s);
    else
        e = weight_dtype == LOOM_SELECT_BF16 ? launch_quant_t<LOOM_SELECT_F32, LOOM_SELECT_BF16, true>(p, sms, s)
                                             : launch_quant_t<LOOM_SELECT_F32, LOOM_SELECT_F32, true>(p, sms, s);
    return e == cudaSuccess ? LOOM_SELECT_OK : LOOM_SELECT_ECUDA;
}

LOOM_SELECT_API int loom_quantize_rows_i8(const void* x, int dtype, int64_t rows, int64_t dim, int64_t x_stride,
                                          int8_t* out_q, float* out_scale, void* stream) {
    if (!dtype_ok(dtype)) return LOOM_SELECT_EDTYPE;
    if (!x || !out_q || !out_scale || rows <= 0 || dim <= 0 || x_stride < dim) return LOOM_SELECT_EINVAL;
    if (misaligned(x, esz_of(dtype)) || misaligned(out_scale, 4)) return LOOM_SELECT_EINVAL;
    if (dim > kMaxDim || rows > INT32_MAX) return LOOM_SELECT_ESHAPE;
    QuantDev p{};
    p.x = static_cast<const unsigned char*>(x);
    p.q = out_q;
    p.scale = out_scale;
    p.rows = rows;
    p.x_stride = x_stride;
    p.dim = int32_t(dim);
    int st = LOOM_SELECT_OK;
    const int sms = device_sm_count(&st);
    if (st != LOOM_SELECT_OK) return st;
    const auto s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == LOOM_SELECT_BF16 ? launch_quant_t<LOOM_SELECT_BF16, LOOM_SELECT_F32, false>(p, sms, s)
                                                    : launch_quant_t<LOOM_SELECT_F32, LOOM_SELECT_F32, false>(p, sms, s);
    return e == cudaSuccess ? LOOM_SELECT_OK : LOOM_SELECT_ECUDA;
}

}  // extern "C"
