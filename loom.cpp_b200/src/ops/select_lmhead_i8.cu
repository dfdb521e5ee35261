// select_lmhead_i8.cu -- the LM-head product on 8-bit integers (sm_100a: TMA + tcgen05 + TMEM).
//
//   logits[r, v] = (f32(sum_k hidden[r, k] * weight[v, k]) * hidden_scale[r]) * weight_scale[v]
//
// with int8 operands, a scale per hidden row (token) and per weight row (vocabulary id). The integer sum is
// exact (32 bits: 128 * 128 * 65536 < 2^31), so a logit has three f32 roundings whatever the order of the
// sum, and a fourth where bf16 logits are asked for.
//
// The weight is the MMA's A operand, 128 ids to a CTA's tile, and the hidden rows its B operand, NR rows to a tile: an
// accumulator lane is an id and its columns are rows, so that a warp's store of one column covers 32 neighbouring ids of
// one row whatever the alignment of the output, and a call of few rows has a narrow MMA and few columns to drain. One
// persistent CTA per SM. Warp 0 streams 128-byte K slices of both tiles into a shared-memory ring with TMA (128-byte
// swizzle, a K tail filled with zeros), warp 1 issues tcgen05.mma kind::i8 (M 128, N NR, K 32) into one of two TMEM
// accumulators, the other warps drain the other one, scale it and write the logits.
// Copies and products are issued by an elected lane: behind `lane == 0` alone the compiler does not know that one thread
// issues, and a slice's four products and their commit took 304 cycles in place of 52, its copies 620 in place of 414
// ([1024, 2048] x [151936, 2048] 262 us, now 230; [1, 8192] x [12000, 8192] 46 and 23).
// Calls of more than 128 rows work in pairs of CTAs (cta_group::2, M 256, N 160 to 256) where they fill the device: each
// loads its own ids and half of the rows, so a stage brings 32 KiB into an SM for the work that a CTA by itself would fetch
// 48 KiB for ([1024, 2048] x [151936, 2048] bf16 logits 230 us, by single CTAs 263).
// With one tile of rows, each CTA (or pair) takes an equal share of the ids, to 16 (a TMA box): 151936 ids are 1187.0
// tiles, whose whole ones would leave 3 of 148 SMs a ninth. With several, they take whole tiles, rows fastest, so that
// those running together share a weight tile through L2.
// Bound: few rows, HBM (the weight, read once); many rows, the tensor cores and the logits' write.
//
// Waits are bounded and wind down as in select_lmhead.cu; a CTA of a pair whose wait runs out leaves the other's to run
// out by themselves, and both meet at the cluster barrier before TMEM is freed.
#include <atomic>
#include <cstdint>
#include <cuda_runtime.h>

#include "loom_select.h"
#include "select_device.cuh"
#include "select_internal.h"
#include "select_tcgen05.cuh"

namespace loom_select {
namespace {

constexpr int kIds = 128;      // ids per tile (MMA M)
constexpr int kBK = 128;       // K slice per stage: 128 int8, one swizzle span
constexpr int kUK = 32;        // K per tcgen05.mma (kind::i8)
constexpr int kMaxHidden = 65536;
constexpr int kUnit = 16;      // ids per TMA box where CTAs share the ids out

// NR: hidden rows per tile (MMA N). kPair: two CTAs to a tile.
template <int NR, bool kPair>
struct I8Tile {
    static_assert(NR % 16 == 0 && NR <= 256, "an MMA N for M = 128 or 256");
    static constexpr int kCtas = kPair ? 2 : 1;
    static constexpr int kBRows = NR / kCtas;  // rows a CTA loads
    static constexpr uint32_t kTileABytes = uint32_t(kIds) * kBK;
    static constexpr uint32_t kTileBBytes = uint32_t(kBRows) * kBK;
    static constexpr uint32_t kStageBytes = kTileABytes + kTileBBytes;
    static_assert(kStageBytes % 1024 == 0, "stage alignment");
    // Warp 0 TMA, warp 1 MMA and TMEM, then the epilogue: four warps cover the accumulator's lanes, eight its columns by
    // halves too (four drained a 256-row tile too slowly: [1024, 2048] x [151936, 2048] bf16 logits 256 us before there were pairs).
    static constexpr int kEpiWarps = NR >= 64 ? 8 : 4;
    static constexpr int kThreads = 64 + 32 * kEpiWarps;
    static constexpr int kEpiCols = NR / (kEpiWarps / 4);  // rows a warp drains of a tile, 32 at a time
    static constexpr int kEpiScales = (kEpiCols + 31) / 32 * 32;
    static constexpr uint32_t kScaleBytes = kEpiWarps * kEpiScales * 4;  // their scales, a copy for each warp
    static constexpr int kFit = int((227u * 1024u - 2048u - kScaleBytes) / kStageBytes);
    static constexpr int kStages = kFit < 12 ? kFit : 12;
    static constexpr size_t kSmemBytes = size_t(kStages) * kStageBytes + kScaleBytes + 512 + 1024;
    static constexpr uint32_t kTmemCols = NR <= 16 ? 32 : NR <= 64 ? 128 : NR <= 128 ? 256 : 512;  // two accumulators
    // Instruction descriptor, kind::i8: s32 accumulator (2), signed A and B (1), K-major, N >> 3, M >> 4.
    static constexpr uint32_t kIdesc =
        (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(NR >> 3) << 17) | (uint32_t(kCtas * kIds >> 4) << 24);
};

template <int kStages>
struct I8Bars {
    uint64_t full[kStages];   // TMA -> MMA: a pair's both copies arrive at the even CTA's
    uint64_t empty[kStages];  // MMA -> TMA, in both CTAs of a pair
    uint64_t tfull[2];        // MMA -> epilogue, in both
    uint64_t tempty[2];       // epilogue warps (of both) -> MMA
    uint64_t drain;           // the MMA warp's final commit
    uint32_t tmem_base;
    int abort;
};

struct I8Args {
    int64_t rows, n_vocab;
    int k_blocks;
    int r_tiles;       // tiles along the rows
    int64_t v_tiles;   // tiles along the ids (r_tiles > 1)
    int64_t units;     // ids / kUnit, rounded up (r_tiles == 1)
    const float* row_scale;
    const float* col_scale;
    void* out;
    int64_t out_stride;
    int* status;
};

// The tiles of one CTA (or pair), in order: this CTA's ids [id, id_end), perhaps none, and rows from `row` on.
template <int NR, bool kPair>
struct I8Walk {
    static constexpr int kCtas = kPair ? 2 : 1;
    int64_t id, id_end;
    int64_t tile_end;  // the end of the tile's ids, both CTAs'
    int64_t row;
    uint32_t next, end;  // one tile of rows: units of ids; several: tiles (fewer than 2^31, in 32 bits: a division each)
    __device__ __forceinline__ explicit I8Walk(const I8Args& a) {
        const uint32_t worker = blockIdx.x / kCtas, workers = gridDim.x / kCtas;
        if (a.r_tiles == 1) {
            next = uint32_t(a.units * worker / workers);
            end = uint32_t(a.units * (worker + 1) / workers);
        } else {
            next = worker;
            end = uint32_t(a.v_tiles * a.r_tiles);
        }
    }
    __device__ __forceinline__ bool step(const I8Args& a) {
        if (next >= end) return false;
        int64_t past;
        if (a.r_tiles == 1) {
            constexpr int kUnits = kCtas * kIds / kUnit;
            id = int64_t(next) * kUnit;
            next = next + kUnits < end ? next + kUnits : end;
            past = int64_t(next) * kUnit;
            row = 0;
        } else {
            const uint32_t v = next / uint32_t(a.r_tiles);
            id = int64_t(v) * (kCtas * kIds);
            past = id + kCtas * kIds;
            row = int64_t(next - v * uint32_t(a.r_tiles)) * NR;
            next += gridDim.x / kCtas;
        }
        tile_end = past < a.n_vocab ? past : a.n_vocab;
        if (kPair && blockIdx.x % 2) id += kIds;
        id_end = tile_end < id + kIds ? tile_end : id + kIds;
        return true;
    }
    // TMA boxes of kUnit ids for the CTA whose ids begin at `from`; 0: one box for its whole tile. Where CTAs share the ids
    // out, what is left of a share goes by small boxes (a whole tile by sixteen of them: 96 us for one row, where one
    // box took 61).
    __device__ __forceinline__ int boxes(const I8Args& a, int64_t from, bool& none) const {
        none = tile_end <= from;
        const int64_t left = (tile_end - from + kUnit - 1) / kUnit;
        return none || a.r_tiles > 1 || left >= kIds / kUnit ? 0 : int(left);
    }
};

template <int kOut>
__device__ __forceinline__ void store_logit(void* out, int64_t i, float v) {
    if constexpr (kOut == LOOM_SELECT_BF16) reinterpret_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<float*>(out)[i] = v;
}

// W rows of one id: accumulator bits, the rows' scales (shared memory, 16-byte aligned) and the id's scale; n rows
// exist, at is the first one's place in the output.
template <int kOut, int W>
__device__ __forceinline__ void write_rows(const I8Args& a, const float (&acc)[W], const float* scale, float col_scale,
                                           int64_t at, int n, bool there) {
    float v[W];
#pragma unroll
    for (int j = 0; j < W; j += 4) {
        const float4 s = *reinterpret_cast<const float4*>(scale + j);
        v[j] = __fmul_rn(__fmul_rn(__int2float_rn(__float_as_int(acc[j])), s.x), col_scale);
        v[j + 1] = __fmul_rn(__fmul_rn(__int2float_rn(__float_as_int(acc[j + 1])), s.y), col_scale);
        v[j + 2] = __fmul_rn(__fmul_rn(__int2float_rn(__float_as_int(acc[j + 2])), s.z), col_scale);
        v[j + 3] = __fmul_rn(__fmul_rn(__int2float_rn(__float_as_int(acc[j + 3])), s.w), col_scale);
    }
    if (!there) return;
    if (n >= W) {
#pragma unroll
        for (int j = 0; j < W; ++j, at += a.out_stride) store_logit<kOut>(a.out, at, v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j, at += a.out_stride)
            if (j < n) store_logit<kOut>(a.out, at, v[j]);
    }
}

template <int NR, bool kPair, int kOut>
__global__ void __launch_bounds__(I8Tile<NR, kPair>::kThreads, 1)
    lm_head_logits_i8_kernel(const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_w,
                             const __grid_constant__ CUtensorMap map_unit, const I8Args a) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    using T = I8Tile<NR, kPair>;
    constexpr int kStages = T::kStages;
    constexpr uint32_t kStageBytes = T::kStageBytes;
    float* scales = reinterpret_cast<float*>(smem + size_t(kStages) * kStageBytes);
    I8Bars<kStages>* bars = reinterpret_cast<I8Bars<kStages>*>(smem + size_t(kStages) * kStageBytes + T::kScaleBytes);
    static_assert(sizeof(I8Bars<kStages>) <= 512, "barriers");
    volatile int* abort_flag = &bars->abort;
    const uint32_t rank = kPair ? blockIdx.x % 2 : 0;  // (clusters are neighbouring blocks)

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WaitFault wf = read_wait_fault(a.status);  // the workspace header's test hook: zero for normal callers
    const uint64_t lim = wf.limit_ns;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bars->tfull[b], 1);
            mbar_init(&bars->tempty[b], T::kCtas * T::kEpiWarps);
        }
        mbar_init(&bars->drain, 1);
        bars->abort = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        if constexpr (kPair) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             smem_addr(&bars->tmem_base)),
                         "r"(T::kTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             smem_addr(&bars->tmem_base)),
                         "r"(T::kTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (kPair) cluster_sync_all();  // the other CTA's barriers are there too
    tc_fence_after();
    const uint32_t tmem_base = bars->tmem_base;
    I8Walk<NR, kPair> walk(a);

    if (warp == 0) {
        if (elect_one()) {
            // ---- producer ----
            // (stage and parity are counted along: dividing the slice's number for them cost 60 cycles a slice)
            int64_t kc = 0;
            int s = 0;
            uint32_t round = 0;  // the ring's passes so far, of which the last bit is the parity
            const int64_t withheld = (blockIdx.x == 0 && wf.withhold > 0) ? int64_t(wf.withhold) - 1 : -1;
            bool ok = true;
            while (ok && walk.step(a)) {
                bool none, peer_none = true;
                const int boxes = walk.boxes(a, walk.id, none);
                uint32_t bytes = T::kTileBBytes + (none ? 0u : boxes ? uint32_t(boxes) * kUnit * kBK : T::kTileABytes);
                if (kPair && rank == 0) {  // the odd CTA's copies too
                    const int peer = walk.boxes(a, walk.id + kIds, peer_none);
                    bytes += T::kTileBBytes + (peer_none ? 0u : peer ? uint32_t(peer) * kUnit * kBK : T::kTileABytes);
                }
                for (int kb = 0; kb < a.k_blocks; ++kb, ++kc, s = s + 1 == kStages ? 0 : s + 1, round += s == 0) {
                    if (round > 0 && !lm_wait(&bars->empty[s], (round - 1) & 1, a.status, abort_flag, lim)) {
                        ok = false;
                        break;
                    }
                    if (kc == withheld) continue;  // test hook only: this slice never arrives
                    unsigned char* st = smem + uint32_t(s) * kStageBytes;
                    if (rank == 0) mbar_arrive_expect_tx(&bars->full[s], bytes);
                    auto load = [&](void* to, const CUtensorMap* map, int64_t y) {
                        if constexpr (kPair) tma_load_2d_pair(to, map, kb * kBK, int(y), &bars->full[s]);
                        else tma_load_2d(to, map, kb * kBK, int(y), &bars->full[s]);
                    };
                    if (!none && boxes == 0) load(st, &map_w, walk.id);
                    for (int u = 0; u < boxes; ++u) load(st + u * kUnit * kBK, &map_unit, walk.id + u * kUnit);
                    load(st + T::kTileABytes, &map_h, walk.row + int(rank) * T::kBRows);
                }
            }
            // Every copy issued lands before the CTA may exit (a withheld slice was never issued). A pair's odd CTA learns it
            // from the MMAs that have read them; where those no longer come, its wait's limit is thousands of copies long.
            for (int t = 0; t < kStages; ++t) {
                // the last pass in which stage t was used: this one, or the one before
                int64_t pass = int64_t(round) - (t < s ? 0 : 1);
                if (withheld >= 0 && pass * kStages + t == withheld) --pass;
                if (pass >= 0)
                    mbar_wait_bounded(rank == 0 ? &bars->full[t] : &bars->empty[t], uint32_t(pass & 1), a.status, lim);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {  // (of a pair, the even CTA's)
            // ---- MMA issuer ----
            int i = 0, s = 0;
            uint32_t parity = 0;
            bool ok = true;
            const uint64_t desc_a = smem_desc_sw128(smem_addr(smem)), desc_b = smem_desc_sw128(smem_addr(smem) + T::kTileABytes);
            for (; ok && walk.step(a); ++i) {
                const int b = i & 1, u = i >> 1;
                if (u >= 1 && !lm_wait(&bars->tempty[b], uint32_t((u - 1) & 1), a.status, abort_flag, lim)) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + uint32_t(b * NR);
                for (int kb = 0; kb < a.k_blocks; ++kb) {
                    if (!lm_wait(&bars->full[s], parity, a.status, abort_flag, lim)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t at = uint32_t(s) * (kStageBytes >> 4);  // (descriptors hold the address's bits from 4 on)
#pragma unroll
                    for (int kk = 0; kk < kBK / kUK; ++kk) {
                        const uint64_t da = desc_a + at + (kk * kUK >> 4), db = desc_b + at + (kk * kUK >> 4);
                        if constexpr (kPair) tc_mma_i8_pair(d_tmem, da, db, T::kIdesc, (kb | kk) != 0 ? 1u : 0u);
                        else tc_mma_i8(d_tmem, da, db, T::kIdesc, (kb | kk) != 0 ? 1u : 0u);
                    }
                    if constexpr (kPair) tc_commit_both(&bars->empty[s]);
                    else tc_commit(&bars->empty[s]);
                    if (++s == kStages) {
                        s = 0;
                        parity ^= 1;
                    }
                }
                if (ok) {
                    if constexpr (kPair) tc_commit_both(&bars->tfull[b]);
                    else tc_commit(&bars->tfull[b]);
                }
            }
            // all MMAs issued have completed before TMEM is freed
            if constexpr (kPair) tc_commit_pair_own(&bars->drain);
            else tc_commit(&bars->drain);
            mbar_wait_bounded(&bars->drain, 0, a.status, lim);
        }
        __syncwarp();
    } else {
        // ---- epilogue: a warp reads TMEM lanes 32 * (warp % 4) .. + 31, one id per thread ----
        const int q = warp & 3, col0 = (warp - 2) / 4 * T::kEpiCols;
        float* scale = scales + (warp - 2) * T::kEpiScales;
        int64_t scale_row = -1;  // the tile whose scales are in `scale`
        for (int i = 0; walk.step(a); ++i) {
            const int b = i & 1, u = i >> 1;
            const int64_t row = walk.row + col0;  // this warp's first
            if (walk.row != scale_row) {
                scale_row = walk.row;
                __syncwarp();
                for (int j = lane; j < T::kEpiScales; j += 32) scale[j] = row + j < a.rows ? __ldg(a.row_scale + row + j) : 0.0f;
                __syncwarp();
            }
            const int64_t id = walk.id + q * 32 + lane;
            const bool there = id < walk.id_end;
            const float col_scale = there ? __ldg(a.col_scale + id) : 0.0f;
            const int n_rows = a.rows - row < T::kEpiCols ? int(a.rows - row) : T::kEpiCols;  // (none: not positive)
            const bool ok = lm_wait(&bars->tfull[b], uint32_t(u & 1), a.status, abort_flag, lim);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            const uint32_t taddr = tmem_base + (uint32_t(q * 32) << 16) + uint32_t(b * NR + col0);
            if (__any_sync(0xffffffffu, there)) {
                int64_t at = row * a.out_stride + id;
                if constexpr (NR < 32) {
                    float v[16];
                    tc_ld16(taddr, v);
                    write_rows<kOut, 16>(a, v, scale, col_scale, at, n_rows, there);
                } else {
#pragma unroll 1
                    for (int c = 0; c < T::kEpiCols && c < n_rows; c += 32, at += 32 * a.out_stride) {
                        float v[32];
                        tc_ld32(taddr + uint32_t(c), v);
                        write_rows<kOut, 32>(a, v, scale + c, col_scale, at, n_rows - c, there);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (kPair && rank != 0) mbar_arrive_remote(&bars->tempty[b], 0);
                else mbar_arrive(&bars->tempty[b]);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    // (neither CTA of a pair leaves, or frees TMEM, while the other may still write to it)
    if constexpr (kPair) cluster_sync_all();
    tc_fence_after();
    if (warp == 1) {
        if constexpr (kPair)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(T::kTmemCols) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(T::kTmemCols) : "memory");
    }
}

template <int NR, bool kPair, int kOut>
int launch_i8(const void* hidden, const void* weight, I8Args a, int64_t hidden_dim, int sms, cudaStream_t stream) {
    using T = I8Tile<NR, kPair>;
    a.r_tiles = int((a.rows + NR - 1) / NR);
    a.v_tiles = (a.n_vocab + T::kCtas * kIds - 1) / (T::kCtas * kIds);
    a.units = (a.n_vocab + kUnit - 1) / kUnit;
    const int64_t work = a.r_tiles == 1 ? a.units : a.v_tiles * a.r_tiles;
    CUtensorMap map_h, map_w, map_unit;
    if (!make_map(&map_h, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, hidden, uint64_t(hidden_dim), uint64_t(a.rows), T::kBRows) ||
        !make_map(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, weight, uint64_t(hidden_dim), uint64_t(a.n_vocab), kIds) ||
        !make_map(&map_unit, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, weight, uint64_t(hidden_dim), uint64_t(a.n_vocab), kUnit))
        return LOOM_SELECT_ECUDA;
    static std::atomic<bool> configured[64] = {};  // set once per device, from any host thread
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return LOOM_SELECT_ECUDA;
    auto kernel = lm_head_logits_i8_kernel<NR, kPair, kOut>;
    if (!configured[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(T::kSmemBytes)) != cudaSuccess)
            return LOOM_SELECT_ECUDA;
        configured[dev] = true;
    }
    const int64_t most = sms / T::kCtas;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned((work < most ? work : most) * T::kCtas));
    cfg.blockDim = dim3(T::kThreads);
    cfg.dynamicSmemBytes = T::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = unsigned(T::kCtas);
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, map_h, map_w, map_unit, a) == cudaSuccess ? LOOM_SELECT_OK : LOOM_SELECT_ECUDA;
}

template <int kOut>
int launch_i8_any(const void* hidden, const void* weight, const I8Args& a, int64_t hidden_dim, int sms,
                  cudaStream_t stream) {
    if (a.rows <= 16) return launch_i8<16, false, kOut>(hidden, weight, a, hidden_dim, sms, stream);
    if (a.rows <= 64) return launch_i8<64, false, kOut>(hidden, weight, a, hidden_dim, sms, stream);
    if (a.rows <= 128) return launch_i8<128, false, kOut>(hidden, weight, a, hidden_dim, sms, stream);
    // a tile for each CTA at most: by themselves, 64 rows a tile if there are CTAs for them ([500, 8192] x [1000, 8192] 17.0
    // us, in pairs 24.7; [200, 8192] x [4000, 8192] 17.4 and 25.4; [500, 8192] x [4000, 8192] of 128 rows 19.6 and 25.4)
    const int64_t v_tiles = (a.n_vocab + kIds - 1) / kIds;
    if ((a.rows + 63) / 64 * v_tiles <= sms) return launch_i8<64, false, kOut>(hidden, weight, a, hidden_dim, sms, stream);
    if ((a.rows + 127) / 128 * v_tiles <= sms) return launch_i8<128, false, kOut>(hidden, weight, a, hidden_dim, sms, stream);
    // as few tiles of rows as there have to be, no higher than they have to be
    const int64_t tiles = (a.rows + 255) / 256, high = (a.rows + tiles - 1) / tiles;
    if (high <= 160) return launch_i8<160, true, kOut>(hidden, weight, a, hidden_dim, sms, stream);
    if (high <= 192) return launch_i8<192, true, kOut>(hidden, weight, a, hidden_dim, sms, stream);
    if (high <= 224) return launch_i8<224, true, kOut>(hidden, weight, a, hidden_dim, sms, stream);
    return launch_i8<256, true, kOut>(hidden, weight, a, hidden_dim, sms, stream);
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
    if ((rows + 255) / 256 * ((n_vocab + kIds - 1) / kIds) > INT32_MAX) return LOOM_SELECT_ESHAPE;
    if (!workspace || workspace_bytes < kWsAlign || reinterpret_cast<uintptr_t>(workspace) % kWsAlign != 0)
        return LOOM_SELECT_EWORKSPACE;
    int st = LOOM_SELECT_OK;
    const int sms = device_sm_count(&st);
    if (st != LOOM_SELECT_OK) return st;
    I8Args a{};
    a.rows = rows;
    a.n_vocab = n_vocab;
    a.k_blocks = int((hidden_dim + kBK - 1) / kBK);
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
