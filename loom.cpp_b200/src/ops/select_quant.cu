// select_quant.cu -- rows to 8-bit integers with a scale per row: behind the final RMS norm, or as they are.
//
// rms_norm_i8, per row, with D = dim:
//   h = x + r          one rounding to the rows' type (stored to out_sum where asked for; h = x without r)
//   inv = 1 / sqrt(sum h^2 / D + eps)      in 64 bits, rounded once to f32
//   y = (h * inv) * w                      two f32 roundings
//   a = max |y|,  scale = a / 127,  q = rint(y * ((1 / a) * 127))      each step one f32 rounding, |q| <= 127
// quantize_rows_i8 takes y = x. The sum of squares is held in 64 bits so that the result does not depend on
// the order of the summation: f32 squares are exact there up to 2^-53, and the one rounding of inv to f32
// comes out the same for any order but for about one row in 10^8. q is then the same bit for bit whatever
// the launch shape, as the plain definition gives it.
// Bound: HBM (rows read once: a thread keeps its elements in registers between the passes).
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

template <int kDtype>
__device__ __forceinline__ float round_to(float v) {
    if constexpr (kDtype == LOOM_SELECT_BF16) return __bfloat162float(__float2bfloat16_rn(v));
    else return v;
}

template <int kDtype>
__device__ __forceinline__ float plain_load(const void* base, int64_t i) {
    if constexpr (kDtype == LOOM_SELECT_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[i]);
    else return reinterpret_cast<const float*>(base)[i];
}

template <int kDtype>
__device__ __forceinline__ void plain_store(void* base, int64_t i, float v) {
    if constexpr (kDtype == LOOM_SELECT_BF16) reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<float*>(base)[i] = v;
}

// kNT threads hold one row, kPer elements each: thread t the elements t, t + kNT, ...
template <int kDtype, int kWDtype, bool kNorm, int kNT, int kPer>
__global__ void __launch_bounds__(kNT) quant_rows_kernel(const QuantDev p) {
    constexpr int kEsz = kDtype == LOOM_SELECT_BF16 ? 2 : 4;
    constexpr int kWarps = kNT / 32;
    __shared__ double part_ss[kWarps];
    __shared__ float part_max[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x;
    const unsigned char* x = p.x + row * p.x_stride * kEsz;
    float h[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = j * kNT + tid;
        h[j] = i < p.dim ? plain_load<kDtype>(x, i) : 0.0f;
    }
    if constexpr (kNorm) {
        if (p.residual) {
            const unsigned char* r = p.residual + row * p.residual_stride * kEsz;
            unsigned char* s = p.sum ? p.sum + row * p.sum_stride * kEsz : nullptr;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const int i = j * kNT + tid;
                if (i < p.dim) {
                    h[j] = round_to<kDtype>(__fadd_rn(h[j], plain_load<kDtype>(r, i)));
                    if (s) plain_store<kDtype>(s, i, h[j]);
                }
            }
        }
        double ss = 0.0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) ss = __fma_rn(double(h[j]), double(h[j]), ss);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (lane == 0) part_ss[warp] = ss;
        __syncthreads();
        ss = part_ss[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) ss += part_ss[w];
        const float inv = __double2float_rn(__drcp_rn(__dsqrt_rn(__ddiv_rn(ss, double(p.dim)) + p.eps)));
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int i = j * kNT + tid;
            if (i < p.dim) h[j] = __fmul_rn(__fmul_rn(h[j], inv), plain_load<kWDtype>(p.weight, i));
        }
    }
    float a = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) a = nan_max(a, fabsf(h[j]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = nan_max(a, __shfl_xor_sync(0xffffffffu, a, o));
    if (lane == 0) part_max[warp] = a;
    __syncthreads();
    a = part_max[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) a = nan_max(a, part_max[w]);
    // a NaN or an infinity anywhere: q 0 and a NaN scale, so that what is made of them is NaN
    const bool fine = a <= FLT_MAX, some = fine && a >= kTinyRow;
    const float inv_scale = some ? __fmul_rn(__frcp_rn(a), 127.0f) : 0.0f;
    if (tid == 0) p.scale[row] = !fine ? __int_as_float(0x7fc00000) : some ? __fdiv_rn(a, 127.0f) : 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = j * kNT + tid;
        if (i < p.dim)
            p.q[row * p.dim + i] = some ? static_cast<int8_t>(__float2int_rn(__fmul_rn(h[j], inv_scale))) : int8_t(0);
    }
}

template <int kDtype, int kWDtype, bool kNorm>
cudaError_t launch_quant_t(const QuantDev& p, cudaStream_t s) {
    const unsigned grid = unsigned(p.rows);
    if (p.dim <= 1024) quant_rows_kernel<kDtype, kWDtype, kNorm, 128, 8><<<grid, 128, 0, s>>>(p);
    else if (p.dim <= 8192) quant_rows_kernel<kDtype, kWDtype, kNorm, 512, 16><<<grid, 512, 0, s>>>(p);
    else quant_rows_kernel<kDtype, kWDtype, kNorm, 1024, 32><<<grid, 1024, 0, s>>>(p);
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
    const auto s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (dtype == LOOM_SELECT_BF16)
        e = weight_dtype == LOOM_SELECT_BF16 ? launch_quant_t<LOOM_SELECT_BF16, LOOM_SELECT_BF16, true>(p, s)
                                             : launch_quant_t<LOOM_SELECT_BF16, LOOM_SELECT_F32, true>(p, s);
    else
        e = weight_dtype == LOOM_SELECT_BF16 ? launch_quant_t<LOOM_SELECT_F32, LOOM_SELECT_BF16, true>(p, s)
                                             : launch_quant_t<LOOM_SELECT_F32, LOOM_SELECT_F32, true>(p, s);
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
    const auto s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == LOOM_SELECT_BF16 ? launch_quant_t<LOOM_SELECT_BF16, LOOM_SELECT_F32, false>(p, s)
                                                    : launch_quant_t<LOOM_SELECT_F32, LOOM_SELECT_F32, false>(p, s);
    return e == cudaSuccess ? LOOM_SELECT_OK : LOOM_SELECT_ECUDA;
}

}  // extern "C"
