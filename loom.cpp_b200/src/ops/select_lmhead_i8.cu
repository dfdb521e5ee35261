// select_lmhead_i8.cu -- the LM-head product on 8-bit integers (sm_100a: TMA + tcgen05 + TMEM).
//
//   logits[r, v] = (f32(sum_k hidden[r, k] * weight[v, k]) * hidden_scale[r]) * weight_scale[v]
//
// with int8 operands, a scale per hidden row (token) and per weight row (vocabulary id). The integer sum is
// exact (32 bits: 128 * 128 * 65536 < 2^31), so a logit has three f32 roundings whatever the order of the
// sum, and a fourth where bf16 logits are asked for. Same plan as the bf16 head (select_lmhead.cu): one persistent
// CTA per SM walks 128-row x BN-id tiles, row tile fastest; warp 0 streams 128-byte K slices of both tiles into a
// shared-memory ring with TMA (128-byte swizzle, a K tail filled with zeros), warp 1 issues tcgen05.mma kind::i8
// (M 128, N BN, K 32) into one of two TMEM accumulators, warps 2-5 drain the other one, scale it and write
// the logits. A warp's 32 x 32 block goes through shared memory so that each store instruction covers 32
// neighbouring ids of one row, whatever the alignment of the output rows.
// Bound: few rows, HBM (the weight, read once); many rows, the tensor cores and the logits' write.
//
// Waits are bounded and wind down as in select_lmhead.cu.
#include <atomic>
#include <cstdint>
#include <cuda_runtime.h>

#include "loom_select.h"
#include "select_device.cuh"
#include "select_internal.h"
#include "select_tcgen05.cuh"

namespace loom_select {
namespace {

constexpr int kBM = 128;       // rows per tile (MMA M)
constexpr int kBK = 128;       // K slice per stage: 128 int8, one swizzle span
constexpr int kUK = 32;        // K per tcgen05.mma (kind::i8)
constexpr int kThreads = 192;  // warp 0 TMA, warp 1 MMA + TMEM owner, warps 2-5 epilogue
constexpr uint32_t kTmemCols = 512;
constexpr int kAccStride = 256;
constexpr int kMaxHidden = 65536;
constexpr int kBufStride = 33;  // floats between rows of a warp's transposing block: no bank conflicts
constexpr uint32_t kEpiBytes = 4 * 32 * kBufStride * 4;

// kFewRows (calls of at most 16 rows): a 16-row hidden tile, as in select_lmhead.cu: the MMA reads 128
// rows of A, and the TMEM lanes of the rows that do not exist are never read.
template <int BN, bool kFewRows>
struct I8Tile {
    static constexpr int kARows = kFewRows ? 16 : kBM;
    static constexpr uint32_t kTileABytes = uint32_t(kARows) * kBK;
    static constexpr uint32_t kTileBBytes = uint32_t(BN) * kBK;
    static constexpr uint32_t kStageBytes = kTileABytes + kTileBBytes;
    static_assert(kStageBytes % 1024 == 0, "stage alignment");
    static constexpr int kFit = int((227u * 1024u - 2048u - kEpiBytes) / kStageBytes);
    static constexpr int kStages = kFit < 8 ? kFit : 8;
    static_assert(kStages >= 2 && kStageBytes >= kBM * kBK, "the MMA's 128-row A read stays inside its stage");
    static constexpr size_t kSmemBytes = size_t(kStages) * kStageBytes + kEpiBytes + 256 + 1024;
    // Instruction descriptor, kind::i8: s32 accumulator (2), signed A and B (1), K-major, N >> 3, M >> 4.
    static constexpr uint32_t kIdesc =
        (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(BN >> 3) << 17) | (uint32_t(kBM >> 4) << 24);
};

struct I8Args {
    int64_t rows, n_vocab;
    int k_blocks;
    int m_tiles, v_tiles;
    const float* row_scale;
    const float* col_scale;
    void* out;
    int64_t out_stride;
    int* status;
};

template <int kOut>
__device__ __forceinline__ void store_logit(void* out, int64_t i, float v) {
    if constexpr (kOut == LOOM_SELECT_BF16) reinterpret_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<float*>(out)[i] = v;
}

// W accumulator columns of the warp's 32 rows, scaled and written: col is the first one's id, n of them
// exist; row0 is lane 0's row, n_rows of the warp's rows exist.
template <int kOut, int W>
__device__ __forceinline__ void write_block(const I8Args& a, float* buf, const float (&acc)[W], float row_scale,
                                            int64_t row0, int n_rows, int64_t col, int n) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < W; ++j) buf[lane * kBufStride + j] = __fmul_rn(__int2float_rn(__float_as_int(acc[j])), row_scale);
    __syncwarp();
    if (lane < n && lane < W) {
        const float cs = __ldg(a.col_scale + col + lane);
        int64_t at = row0 * a.out_stride + col + lane;
        for (int r = 0; r < n_rows; ++r, at += a.out_stride)
            store_logit<kOut>(a.out, at, __fmul_rn(buf[r * kBufStride + lane], cs));
    }
    __syncwarp();
}

template <int BN, bool kFewRows, int kOut>
__global__ void __launch_bounds__(kThreads, 1)
    lm_head_logits_i8_kernel(const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_w,
                             const I8Args a) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    using T = I8Tile<BN, kFewRows>;
    constexpr uint32_t kTileABytes = T::kTileABytes;
    constexpr int kStages = T::kStages;
    constexpr uint32_t kStageBytes = T::kStageBytes;
    float* epi = reinterpret_cast<float*>(smem + size_t(kStages) * kStageBytes);
    LmBars<kStages>* bars = reinterpret_cast<LmBars<kStages>*>(smem + size_t(kStages) * kStageBytes + kEpiBytes);
    volatile int* abort_flag = &bars->abort;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WaitFault wf = read_wait_fault(a.status);  // the workspace header's test hook: zero for normal callers
    const uint64_t lim = wf.limit_ns;
    const int n_tiles = a.m_tiles * a.v_tiles;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bars->tfull[b], 1);
            mbar_init(&bars->tempty[b], 4);
        }
        mbar_init(&bars->drain, 1);
        bars->abort = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&bars->tmem_base)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = bars->tmem_base;

    if (warp == 0) {
        if (lane == 0) {
            // ---- producer ----
            int64_t kc = 0;
            const int64_t withheld = (blockIdx.x == 0 && wf.withhold > 0) ? int64_t(wf.withhold) - 1 : -1;
            bool ok = true;
            for (int t = blockIdx.x; t < n_tiles && ok; t += gridDim.x) {
                const int mt = t % a.m_tiles, vt = t / a.m_tiles;
                for (int kb = 0; kb < a.k_blocks; ++kb, ++kc) {
                    const int s = int(kc % kStages);
                    const int64_t n = kc / kStages;
                    if (n >= 1 && !lm_wait(&bars->empty[s], uint32_t((n - 1) & 1), a.status, abort_flag, lim)) {
                        ok = false;
                        break;
                    }
                    if (kc == withheld) continue;  // test hook only: this slice never arrives
                    unsigned char* st = smem + size_t(s) * kStageBytes;
                    mbar_arrive_expect_tx(&bars->full[s], kStageBytes);
                    tma_load_2d(st, &map_h, kb * kBK, mt * kBM, &bars->full[s]);
                    tma_load_2d(st + kTileABytes, &map_w, kb * kBK, vt * BN, &bars->full[s]);
                }
            }
            // every copy issued lands before the CTA may exit (a withheld slice was never issued)
            for (int s = 0; s < kStages; ++s) {
                if (kc > s) {
                    int64_t last_kc = s + int64_t(kStages) * ((kc - 1 - s) / kStages);
                    if (last_kc == withheld) last_kc -= kStages;
                    if (last_kc >= 0) mbar_wait_bounded(&bars->full[s], uint32_t((last_kc / kStages) & 1), a.status, lim);
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            // ---- MMA issuer ----
            int64_t kc = 0;
            int i = 0;
            bool ok = true;
            for (int t = blockIdx.x; t < n_tiles && ok; t += gridDim.x, ++i) {
                const int b = i & 1, u = i >> 1;
                if (u >= 1 && !lm_wait(&bars->tempty[b], uint32_t((u - 1) & 1), a.status, abort_flag, lim)) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + uint32_t(b * kAccStride);
                for (int kb = 0; kb < a.k_blocks; ++kb, ++kc) {
                    const int s = int(kc % kStages);
                    const int64_t n = kc / kStages;
                    if (!lm_wait(&bars->full[s], uint32_t(n & 1), a.status, abort_flag, lim)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sa = smem_addr(smem + size_t(s) * kStageBytes);
                    const uint32_t sb = sa + kTileABytes;
#pragma unroll
                    for (int kk = 0; kk < kBK / kUK; ++kk) {
                        tc_mma_i8(d_tmem, smem_desc_sw128(sa + kk * kUK), smem_desc_sw128(sb + kk * kUK), T::kIdesc,
                                  (kb | kk) != 0 ? 1u : 0u);
                    }
                    tc_commit(&bars->empty[s]);
                }
                if (ok) tc_commit(&bars->tfull[b]);
            }
            // all MMAs issued have completed before TMEM is freed
            tc_commit(&bars->drain);
            mbar_wait_bounded(&bars->drain, 0, a.status, lim);
        }
        __syncwarp();
    } else {
        // ---- epilogue: warps 2-5 read TMEM lanes 32 * (warp % 4) .. + 31, one row per thread ----
        const int q = warp & 3;
        float* buf = epi + q * 32 * kBufStride;
        int i = 0;
        for (int t = blockIdx.x; t < n_tiles; t += gridDim.x, ++i) {
            const int mt = t % a.m_tiles, vt = t / a.m_tiles;
            const int b = i & 1, u = i >> 1;
            const int64_t row0 = int64_t(mt) * kBM + q * 32;
            const int n_rows = a.rows - row0 < 32 ? (a.rows > row0 ? int(a.rows - row0) : 0) : 32;
            const float row_scale = lane < n_rows ? __ldg(a.row_scale + row0 + lane) : 0.0f;
            const bool ok = lm_wait(&bars->tfull[b], uint32_t(u & 1), a.status, abort_flag, lim);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            if (n_rows > 0) {
                const uint32_t taddr = tmem_base + (uint32_t(q * 32) << 16) + uint32_t(b * kAccStride);
                const int64_t col0 = int64_t(vt) * BN;
                const int valid = a.n_vocab - col0 < BN ? int(a.n_vocab - col0) : BN;
                constexpr int kFull = BN / 32 * 32;
#pragma unroll 1
                for (int c = 0; c < kFull; c += 32) {
                    float v[32];
                    tc_ld32(taddr + uint32_t(c), v);
                    write_block<kOut, 32>(a, buf, v, row_scale, row0, n_rows, col0 + c, valid - c);
                }
                if constexpr (BN % 32 != 0) {
                    float w[16];
                    tc_ld16(taddr + uint32_t(kFull), w);
                    write_block<kOut, 16>(a, buf, w, row_scale, row0, n_rows, col0 + kFull, valid - kFull);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->tempty[b]);
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
    }
}

bool make_map_i8(CUtensorMap* m, const void* base, uint64_t inner, uint64_t outer, uint32_t box_outer) {
    auto fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {inner, outer};
    const cuuint64_t strides[1] = {inner};
    const cuuint32_t box[2] = {uint32_t(kBK), box_outer};
    const cuuint32_t estr[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tile widths, chosen as in the bf16 head: 208 ids where that spreads the tiles over the SMs clearly more
// evenly (151936 ids on one row tile: 594 tiles of 256 leave two SMs a fifth tile).
constexpr int kWideBN = 256, kNarrowBN = 208;

int pick_bn(int64_t m_tiles, int64_t n_vocab, int sms) {
    auto cost = [&](int bn) {
        const int64_t tiles = m_tiles * ((n_vocab + bn - 1) / bn);
        return double((tiles + sms - 1) / sms) * bn;
    };
    return cost(kNarrowBN) < 0.97 * cost(kWideBN) ? kNarrowBN : kWideBN;
}

template <int BN, bool kFewRows, int kOut>
int launch_i8(const void* hidden, const void* weight, I8Args a, int64_t hidden_dim, int sms, cudaStream_t stream) {
    using T = I8Tile<BN, kFewRows>;
    a.v_tiles = int((a.n_vocab + BN - 1) / BN);
    CUtensorMap map_h, map_w;
    if (!make_map_i8(&map_h, hidden, uint64_t(hidden_dim), uint64_t(a.rows), uint32_t(T::kARows)) ||
        !make_map_i8(&map_w, weight, uint64_t(hidden_dim), uint64_t(a.n_vocab), BN))
        return LOOM_SELECT_ECUDA;
    static std::atomic<bool> configured[64] = {};  // set once per device, from any host thread
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return LOOM_SELECT_ECUDA;
    if (!configured[dev]) {
        if (cudaFuncSetAttribute(lm_head_logits_i8_kernel<BN, kFewRows, kOut>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, int(T::kSmemBytes)) != cudaSuccess)
            return LOOM_SELECT_ECUDA;
        configured[dev] = true;
    }
    const int64_t tiles = int64_t(a.m_tiles) * a.v_tiles;
    const int grid = int(tiles < sms ? tiles : sms);
    lm_head_logits_i8_kernel<BN, kFewRows, kOut><<<grid, kThreads, T::kSmemBytes, stream>>>(map_h, map_w, a);
    return cudaGetLastError() == cudaSuccess ? LOOM_SELECT_OK : LOOM_SELECT_ECUDA;
}

template <int kOut>
int launch_i8_any(const void* hidden, const void* weight, const I8Args& a, int64_t hidden_dim, int sms,
                  cudaStream_t stream) {
    const bool few = a.rows <= 16;
    if (pick_bn(a.m_tiles, a.n_vocab, sms) == kNarrowBN)
        return few ? launch_i8<kNarrowBN, true, kOut>(hidden, weight, a, hidden_dim, sms, stream)
                   : launch_i8<kNarrowBN, false, kOut>(hidden, weight, a, hidden_dim, sms, stream);
    return few ? launch_i8<kWideBN, true, kOut>(hidden, weight, a, hidden_dim, sms, stream)
               : launch_i8<kWideBN, false, kOut>(hidden, weight, a, hidden_dim, sms, stream);
}

}  // namespace
}  // namespace loom_select

using namespace loom_select;

extern "C" {

LOOM_SELECT_API size_t loom_lm_head_logits_i8_workspace_size(int64_t rows, int64_t n_vocab) {
    (void)rows, (void)n_vocab;
    return kWsAlign;  // the status word
}

LOOM_SELECT_API int loom_lm_head_logits_i8(const int8_t* hidden, const float* hidden_scale, const int8_t* weight,
                                           const float* weight_scale, int64_t rows, int64_t hidden_dim,
                                           int64_t n_vocab, void* out_logits, int out_dtype, int64_t out_stride,
                                           void* workspace, size_t workspace_bytes, void* stream) {
    if (out_dtype != LOOM_SELECT_F32 && out_dtype != LOOM_SELECT_BF16) return LOOM_SELECT_EDTYPE;
    if (!hidden || !hidden_scale || !weight || !weight_scale || !out_logits) return LOOM_SELECT_EINVAL;
    if (rows <= 0 || hidden_dim <= 0 || n_vocab <= 0 || out_stride < n_vocab) return LOOM_SELECT_EINVAL;
    if (hidden_dim % 16 != 0 || hidden_dim > kMaxHidden || rows > INT32_MAX || n_vocab > INT32_MAX)
        return LOOM_SELECT_ESHAPE;
    const size_t osz = out_dtype == LOOM_SELECT_BF16 ? 2 : 4;
    if (reinterpret_cast<uintptr_t>(hidden) % 16 != 0 || reinterpret_cast<uintptr_t>(weight) % 16 != 0 ||
        reinterpret_cast<uintptr_t>(hidden_scale) % 4 != 0 || reinterpret_cast<uintptr_t>(weight_scale) % 4 != 0 ||
        reinterpret_cast<uintptr_t>(out_logits) % osz != 0)
        return LOOM_SELECT_EINVAL;
    const int64_t mt = (rows + kBM - 1) / kBM;
    if (mt * ((n_vocab + kNarrowBN - 1) / kNarrowBN) > INT32_MAX) return LOOM_SELECT_ESHAPE;
    if (!workspace || workspace_bytes < kWsAlign || reinterpret_cast<uintptr_t>(workspace) % kWsAlign != 0)
        return LOOM_SELECT_EWORKSPACE;
    int st = LOOM_SELECT_OK;
    const int sms = device_sm_count(&st);
    if (st != LOOM_SELECT_OK) return st;
    I8Args a;
    a.rows = rows;
    a.n_vocab = n_vocab;
    a.k_blocks = int((hidden_dim + kBK - 1) / kBK);
    a.m_tiles = int(mt);
    a.v_tiles = 0;
    a.row_scale = hidden_scale;
    a.col_scale = weight_scale;
    a.out = out_logits;
    a.out_stride = out_stride;
    a.status = static_cast<int*>(workspace);
    const auto s = static_cast<cudaStream_t>(stream);
    return out_dtype == LOOM_SELECT_BF16 ? launch_i8_any<LOOM_SELECT_BF16>(hidden, weight, a, hidden_dim, sms, s)
                                         : launch_i8_any<LOOM_SELECT_F32>(hidden, weight, a, hidden_dim, sms, s);
}

}  // extern "C"
