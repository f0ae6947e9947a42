// Matrix product in 8-bit floating point (e4m3 x e4m3) with an fp32 scale for each 128 of K and each row of a, and for each
// 128 x 128 of w:
//   y[m][n] = sum_b a_scales[b][m] * w_scales[n / 128][b] * sum_{k in b} a[m][k] * w[n][k]  (+ bias[n])
// The inner sums are tcgen05.mma into TMEM, a block of 128 at a time and two accumulators in turn; while the next block's
// MMAs run, the epilogue warps read the finished one back, scale it and add it to the sums that they hold in registers, in fp32.
#include "ptx_sm100.cuh"
#include "rows_common.cuh"
#include "tensor_map.cuh"

namespace exb {
namespace {

constexpr int kBlk = 128;                  // K block: bytes of a row in a stage, elements that share a scale
constexpr int kTileM = 128, kTileN = 128;
constexpr int kStages = 6;
constexpr int kEpiWarps = 8;               // two per TMEM lane quarter, half of the columns each
constexpr int kThreads = (2 + kEpiWarps) * 32;
constexpr int kStageBytes = (kTileM + kTileN) * kBlk;
constexpr uint32_t kMaxSpins = 1u << 21;

struct MatmulParams {
    CUtensorMap tmA, tmW;
    const float *a_scales, *w_scales, *bias;
    void* y;
    int64_t a_scale_stride, w_scale_stride, y_stride;
    int M, N, blocks, y_dtype;
    uint32_t idesc;
    int* error;
};

__device__ __forceinline__ void store_one(void* y, int dtype, int64_t at, float v) {
    if (dtype == EXB_F16) static_cast<__half*>(y)[at] = __float2half_rn(v);
    else if (dtype == EXB_BF16) static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
    else static_cast<float*>(y)[at] = v;
}

__global__ void __launch_bounds__(kThreads, 1) fp8_matmul_kernel(const __grid_constant__ MatmulParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages], tfull_bar[2], tempty_bar[2];
    __shared__ uint32_t tmem_base_smem;
    __shared__ int abort_flag;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = ptx::uniform_warp(), lane = threadIdx.x & 31;
    const int n0 = blockIdx.x * kTileN, m0 = blockIdx.y * kTileM;
    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(&full_bar[s], 1);
            ptx::mbar_init(&empty_bar[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&tfull_bar[i], 1);
            ptx::mbar_init(&tempty_bar[i], kEpiWarps);
        }
        ptx::fence_mbar_init();
        ptx::tma_prefetch_desc(&p.tmA);
        ptx::tma_prefetch_desc(&p.tmW);
    }
    if (warp == 1) {
        ptx::tmem_alloc(&tmem_base_smem, 2 * kTileN);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_smem, 0);
    const uint32_t ring0 = ptx::smem_u32(ring), full0 = ptx::smem_u32(full_bar), empty0 = ptx::smem_u32(empty_bar);
    const uint32_t tfull0 = ptx::smem_u32(tfull_bar), tempty0 = ptx::smem_u32(tempty_bar);
    pdl_wait();
    if (warp == 0) {
        if (lane == 0) {
            const uint64_t mapA = reinterpret_cast<uint64_t>(&p.tmA), mapW = reinterpret_cast<uint64_t>(&p.tmW);
            bool ok = true;
            for (int b = 0; b < p.blocks; ++b) {
                const int s = b % kStages;
                if (b >= kStages && !ptx::mbar_wait_bounded_u32(empty0 + s * 8, (uint32_t)(b / kStages - 1) & 1u, &abort_flag, kMaxSpins)) {
                    ok = false;
                    break;
                }
                ptx::mbar_arrive_expect_tx_u32(full0 + s * 8, kStageBytes);
                ptx::tma_load_2d_u32(ring0 + s * kStageBytes, mapA, full0 + s * 8, b * kBlk, m0);
                ptx::tma_load_2d_u32(ring0 + s * kStageBytes + kTileM * kBlk, mapW, full0 + s * 8, b * kBlk, n0);
            }
            if (!ok) ptx::give_up(p.error, 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        const uint32_t leader = ptx::elect_one() ? 1u : 0u;
        const uint64_t d0 = ptx::make_smem_desc(ring0, kBlk);
        const uint32_t desc_hi = (uint32_t)(d0 >> 32);
        bool ok = true;
        for (int b = 0; b < p.blocks; ++b) {
            const int s = b % kStages, buf = b & 1;
            if ((b >= 2 && !ptx::mbar_wait_bounded_uniform(tempty0 + buf * 8, (uint32_t)(b / 2 - 1) & 1u, &abort_flag, kMaxSpins)) ||
                !ptx::mbar_wait_bounded_uniform(full0 + s * 8, (uint32_t)(b / kStages) & 1u, &abort_flag, kMaxSpins)) {
                ok = false;
                break;
            }
            ptx::tc_fence_after_sync();
            const uint32_t a_lo = (uint32_t)d0 + ((uint32_t)(s * kStageBytes) >> 4), w_lo = a_lo + ((kTileM * kBlk) >> 4);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
                ptx::tc_mma_f8<false>(tmem_base + buf * kTileN, a_lo + 2 * ks, w_lo + 2 * ks, desc_hi, p.idesc, ks ? 1u : 0u, leader);
            if (b + kStages < p.blocks) ptx::tc_commit_u32(empty0 + s * 8, leader);
            ptx::tc_commit_u32(tfull0 + buf * 8, leader);
        }
        if (!ok) ptx::give_up(p.error, 2);
        __syncwarp();
    } else {
        const int q = warp & 3, half = warp < 6 ? 0 : 1, row = m0 + q * 32 + lane, col = n0 + half * 64;
        float acc[64];
#pragma unroll
        for (int i = 0; i < 64; ++i) acc[i] = 0.f;
        bool ok = true;
        for (int b = 0; b < p.blocks; ++b) {
            const int buf = b & 1;
            const float s = row < p.M ? __ldg(p.a_scales + (int64_t)b * p.a_scale_stride + row) * __ldg(p.w_scales + (int64_t)(n0 / kBlk) * p.w_scale_stride + b) : 0.f;
            if (!ptx::mbar_wait_bounded_uniform(tfull0 + buf * 8, (uint32_t)(b / 2) & 1u, &abort_flag, kMaxSpins)) {
                ok = false;
                break;
            }
            __syncwarp();
            ptx::tc_fence_after_sync();
            const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * kTileN + half * 64);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t raw[16];
                ptx::tmem_ld_32x32b_x16(taddr + i * 16, raw);
                ptx::tmem_ld_wait(raw);
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[i * 16 + j] = fmaf(__uint_as_float(raw[j]), s, acc[i * 16 + j]);
            }
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_u32(tempty0 + buf * 8);
        }
        if (!ok && lane == 0) atomicExch(p.error, 3);
        if (ok && row < p.M) {
            const int64_t at = (int64_t)row * p.y_stride + col;
#pragma unroll
            for (int i = 0; i < 64; ++i)
                if (col + i < p.N) store_one(p.y, p.y_dtype, at + i, p.bias ? acc[i] + __ldg(p.bias + col + i) : acc[i]);
        }
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, 2 * kTileN);
    }
}

// ---- CTA pairs ---------------------------------------------------------------------------------
// Tiles of 256 x 256 by pairs of CTAs, persistent.  Each CTA keeps 128 rows of a and half of w's rows of a stage, 32 KB for
// 512 cycles of MMA: 64 bytes per cycle and SM from L2 (a lone CTA's tile of 128 x 128 needs 128).  TMEM holds two accumulators of
// 256 columns; a thread's sums are 128 registers.
constexpr int kPairStages = 6;
constexpr int kPairEpiWarps = 8;                 // two per TMEM lane quarter
constexpr int kPairCols = 4 * 256 / kPairEpiWarps;      // of the accumulator's columns each
constexpr int kPairM = 256, kPairN = 256;
constexpr int kPairStageBytes = (kPairM + kPairN) / 2 * kBlk;      // of one of the two CTAs

struct PairParams {
    CUtensorMap tmA, tmW;
    const float *a_scales, *w_scales, *bias;
    void* y;
    int64_t a_scale_stride, w_scale_stride, y_stride;
    int M, N, blocks, y_dtype, vec;
    int m_tiles, n_tiles;
    uint32_t idesc;
    int* error;
};

// 32 rows x 128 bytes of results per warp, in units of 16 bytes that are XOR-ed with the row: a thread writes its row's units and
// the warp reads whole rows, both without bank conflicts.
constexpr int kStageOut = 32 * 128;

template <typename T>
__device__ __forceinline__ uint32_t result_pair(float a, float b) {
    return rows::float_to_pair(a, b, T());
}

// Columns [col, col + kPairCols) of 32 rows from row0 on: sums in `acc` (a thread has a row), through shared memory to y in full lines.
template <typename T>
__device__ __forceinline__ void store_rows(const float (&acc)[kPairCols], uint8_t* stage, T* y, int64_t y_stride, const float* bias, int row0, int col, int M, int N,
                                           bool vec, int lane) {
    constexpr int kPer = 16 / (int)sizeof(T), kCols = 8 * kPer;      // columns in a unit, in a pass
#pragma unroll
    for (int c0 = 0; c0 < kPairCols; c0 += kCols) {
        if (col + c0 >= N) break;
        const int left = N - col - c0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            float v[kPer];
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[j] = acc[c0 + u * kPer + j];
            if (bias) {
#pragma unroll
                for (int j = 0; j < kPer; ++j)
                    if (u * kPer + j < left) v[j] += __ldg(bias + col + c0 + u * kPer + j);
            }
            uint4 o;
            if constexpr (sizeof(T) == 4)
                o = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
            else
                o = make_uint4(result_pair<T>(v[0], v[1]), result_pair<T>(v[2], v[3]), result_pair<T>(v[4], v[5]), result_pair<T>(v[6], v[7]));
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((u ^ (lane & 7)) << 4)) = o;
        }
        __syncwarp();
        T* out = y + col + c0;
        if (vec && left >= kCols) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = i * 4 + (lane >> 3), u = lane & 7;
                const uint4 o = *reinterpret_cast<const uint4*>(stage + r * 128 + ((u ^ (r & 7)) << 4));
                if (row0 + r < M) *reinterpret_cast<uint4*>(out + (int64_t)(row0 + r) * y_stride + u * kPer) = o;
            }
        } else {
            for (int r = 0; r < 32 && row0 + r < M; ++r) {
#pragma unroll
                for (int c = 0; c < kCols; c += 32) {
                    const int cc = c + lane;
                    const T o = *reinterpret_cast<const T*>(stage + r * 128 + (((cc / kPer) ^ (r & 7)) << 4) + (cc % kPer) * sizeof(T));
                    if (cc < left) out[(int64_t)(row0 + r) * y_stride + cc] = o;
                }
            }
        }
        __syncwarp();
    }
}

// Tiles in an order in which those that run at the same time share rows of a and w: columns of 8 tiles, one after the other.
__device__ __forceinline__ void tile_at(int t, int m_tiles, int n_tiles, int& m, int& n) {
    const int group = t / (8 * n_tiles), first = group * 8, size = min(m_tiles - first, 8);
    const int r = t - group * 8 * n_tiles;
    n = r / size;
    m = first + r - n * size;
}

// Warp 0 loads, warp 1 issues the MMAs, two warpgroups keep the sums: 2 x 224 + 56 registers are the 3 x 168 of the launch.
constexpr int kPairThreads = 128 + kPairEpiWarps * 32;
template <int kRegs> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }

__global__ void __launch_bounds__(kPairThreads, 1) fp8_matmul_pair_kernel(const __grid_constant__ PairParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kPairStages], empty_bar[kPairStages], tfull_bar[2], tempty_bar[2];
    __shared__ uint32_t tmem_base_smem;
    __shared__ int abort_flag;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = ptx::uniform_warp(), lane = threadIdx.x & 31;
    const int rank = (int)__shfl_sync(0xffffffffu, ptx::cluster_ctarank(), 0);
    const int total = p.m_tiles * p.n_tiles, first = blockIdx.x >> 1, step = gridDim.x >> 1;
    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < kPairStages; ++s) {
            ptx::mbar_init(&full_bar[s], 1);
            ptx::mbar_init(&empty_bar[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&tfull_bar[i], 1);
            ptx::mbar_init(&tempty_bar[i], 2 * kPairEpiWarps);      // both CTAs' warps arrive at rank 0
        }
        ptx::fence_mbar_init();
        ptx::tma_prefetch_desc(&p.tmA);
        ptx::tma_prefetch_desc(&p.tmW);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(&tmem_base_smem, 2 * kPairN);
        ptx::tmem_relinquish_pair();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_smem, 0);
    const uint32_t ring0 = ptx::smem_u32(ring), full0 = ptx::smem_u32(full_bar), empty0 = ptx::smem_u32(empty_bar);
    const uint32_t tfull0 = ptx::smem_u32(tfull_bar), tempty0 = ptx::smem_u32(tempty_bar);
    pdl_wait();
    if (warp < 4) {
    fewer_registers<56>();
    if (warp == 0) {
        if (lane == 0) {
            const uint64_t mapA = reinterpret_cast<uint64_t>(&p.tmA), mapW = reinterpret_cast<uint64_t>(&p.tmW);
            const uint32_t full_lead = ptx::map_to_cta(full0, 0);      // both CTAs' bytes are counted by rank 0
            bool ok = true;
            int s = 0;
            uint32_t phase = 1;      // (a fresh barrier's previous phase counts as complete)
            for (int t = first; t < total && ok; t += step) {
                int mt, nt;
                tile_at(t, p.m_tiles, p.n_tiles, mt, nt);
                const int m0 = mt * kPairM + rank * 128, n0 = nt * kPairN + rank * 128;
                for (int b = 0; b < p.blocks; ++b) {
                    if (!ptx::mbar_wait_bounded_u32(empty0 + s * 8, phase, &abort_flag, kMaxSpins)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) ptx::mbar_arrive_expect_tx_u32(full0 + s * 8, 2 * kPairStageBytes);
                    ptx::tma_load_2d_pair(ring0 + s * kPairStageBytes, mapA, full_lead + s * 8, b * kBlk, m0);
                    ptx::tma_load_2d_pair(ring0 + s * kPairStageBytes + 128 * kBlk, mapW, full_lead + s * 8, b * kBlk, n0);
                    if (++s == kPairStages) {
                        s = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (!ok) ptx::give_up(p.error, 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {      // issues for both
            const uint32_t leader = ptx::elect_one() ? 1u : 0u;
            const uint64_t d0 = ptx::make_smem_desc(ring0, kBlk);
            const uint32_t desc_hi = (uint32_t)(d0 >> 32);
            bool ok = true;
            int s = 0, buf = 0;
            uint32_t phase = 0, acc_phase = 1;
            for (int t = first; t < total && ok; t += step) {
                for (int b = 0; b < p.blocks; ++b) {
                    // (the loads are ahead: what is waited for last is what comes last)
                    if (!ptx::mbar_wait_bounded_uniform(full0 + s * 8, phase, &abort_flag, kMaxSpins) ||
                        !ptx::mbar_wait_bounded_uniform(tempty0 + buf * 8, acc_phase, &abort_flag, kMaxSpins)) {
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after_sync();
                    const uint32_t a_lo = (uint32_t)d0 + ((uint32_t)(s * kPairStageBytes) >> 4), w_lo = a_lo + ((128 * kBlk) >> 4);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        ptx::tc_mma_f8<true>(tmem_base + buf * kPairN, a_lo + 2 * ks, w_lo + 2 * ks, desc_hi, p.idesc, ks ? 1u : 0u, leader);
                    ptx::tc_commit_pair_u32(empty0 + s * 8, leader);
                    ptx::tc_commit_pair_u32(tfull0 + buf * 8, leader);
                    if (++s == kPairStages) {
                        s = 0;
                        phase ^= 1u;
                    }
                    if (buf ^= 1; buf == 0) acc_phase ^= 1u;
                }
            }
            if (!ok) ptx::give_up(p.error, 2);
        }
        __syncwarp();
    }
    } else {
        more_registers<224>();
        const int q = warp & 3, part = (warp >> 2) - 1;
        uint8_t* stage = ring + kPairStages * kPairStageBytes + (warp - 4) * kStageOut;
        const uint32_t taddr0 = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(part * kPairCols);
        const uint32_t tempty_lead = ptx::map_to_cta(tempty0, 0);
        bool ok = true;
        int buf = 0;
        uint32_t acc_phase = 0;
        for (int t = first; t < total && ok; t += step) {
            int mt, nt;
            tile_at(t, p.m_tiles, p.n_tiles, mt, nt);
            const int row = mt * kPairM + rank * 128 + q * 32 + lane, col = nt * kPairN + part * kPairCols;
            // this row's and these columns' scales of the next two blocks are on their way while one is worked on
            const float* sa = p.a_scales + (row < p.M ? row : 0);
            const float* sw = p.w_scales + (int64_t)(col < p.N ? col / kBlk : 0) * p.w_scale_stride;
            float sa0 = __ldg(sa), sw0 = __ldg(sw), sa1 = 0.f, sw1 = 0.f;
            if (p.blocks > 1) {
                sa1 = __ldg(sa += p.a_scale_stride);
                sw1 = __ldg(++sw);
            }
            float acc[kPairCols];
#pragma unroll
            for (int i = 0; i < kPairCols; ++i) acc[i] = 0.f;
            for (int b = 0; b < p.blocks; ++b) {
                float sa2 = 0.f, sw2 = 0.f;
                if (b + 2 < p.blocks) {
                    sa2 = __ldg(sa += p.a_scale_stride);
                    sw2 = __ldg(++sw);
                }
                if (!ptx::mbar_wait_bounded_uniform(tfull0 + buf * 8, acc_phase, &abort_flag, kMaxSpins)) {
                    ok = false;
                    break;
                }
                __syncwarp();      // (what follows needs the warp together)
                ptx::tc_fence_after_sync();
                const uint32_t taddr = taddr0 + (uint32_t)(buf * kPairN);
                const float s = sa0 * sw0;
#pragma unroll
                for (int c = 0; c < kPairCols; c += 16) {
                    uint32_t raw[16];
                    ptx::tmem_ld_32x32b_x16(taddr + c, raw);
                    ptx::tmem_ld_wait(raw);
                    if (c + 16 == kPairCols) {
                        ptx::tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) ptx::mbar_arrive_cluster_u32(tempty_lead + buf * 8);
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[c + j] = fmaf(__uint_as_float(raw[j]), s, acc[c + j]);
                }
                sa0 = sa1;
                sw0 = sw1;
                sa1 = sa2;
                sw1 = sw2;
                if (buf ^= 1; buf == 0) acc_phase ^= 1u;
            }
            if (!ok) break;
            const int row0 = row - lane;
            if (p.y_dtype == EXB_F16) store_rows(acc, stage, static_cast<__half*>(p.y), p.y_stride, p.bias, row0, col, p.M, p.N, p.vec, lane);
            else if (p.y_dtype == EXB_BF16) store_rows(acc, stage, static_cast<__nv_bfloat16*>(p.y), p.y_stride, p.bias, row0, col, p.M, p.N, p.vec, lane);
            else store_rows(acc, stage, static_cast<float*>(p.y), p.y_stride, p.bias, row0, col, p.M, p.N, p.vec, lane);
        }
        if (!ok && lane == 0) atomicExch(p.error, 3);
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();      // neither CTA leaves while its peer may still signal its barriers or read its TMEM
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem_base, 2 * kPairN);
    }
}

// Rows of K bytes in boxes of 128 bytes x box_rows, 128-byte swizzle; zeros beyond the matrix.
int encode(CUtensorMap* map, const uint8_t* base, int64_t rows, int K, int64_t stride, int box_rows) {
    const auto fn = tensor_map_encoder();
    if (!fn) return fail(EXB_ERR_CUDA, "exb_fp8_matmul_fwd: the driver has no cuTensorMapEncodeTiled");
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
    cuuint32_t box[2] = {(cuuint32_t)kBlk, (cuuint32_t)box_rows}, step[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(EXB_ERR_CUDA, "exb_fp8_matmul_fwd: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return EXB_OK;
}

}  // namespace
}  // namespace exb

using namespace exb;

extern "C" int exb_fp8_matmul_fwd(exb_ctx* ctx, const uint8_t* a, int64_t a_stride, const float* a_scales, int64_t a_scale_stride,
                                  const uint8_t* w, int64_t w_stride, const float* w_scales, int64_t w_scale_stride, const float* bias, void* y,
                                  int y_dtype, int64_t y_stride, int64_t M, int N, int K, void* stream) {
    EXB_REQUIRE(ctx != nullptr, "exb_fp8_matmul_fwd: null context");
    const size_t es = rows::element_size(y_dtype);
    EXB_REQUIRE(es != 0, "exb_fp8_matmul_fwd: y must be EXB_F16, EXB_BF16 or EXB_F32, got %d", y_dtype);
    EXB_REQUIRE(M >= 0 && N >= 1 && K >= 1, "exb_fp8_matmul_fwd: bad shape (%lld x %d x %d)", (long long)M, N, K);
    if (M > INT32_MAX - 256 || N > INT32_MAX - 256 || K > INT32_MAX - 256)
        return fail(EXB_ERR_UNSUPPORTED, "exb_fp8_matmul_fwd: %lld x %d x %d is too large for one call", (long long)M, N, K);
    if (M == 0) return EXB_OK;
    EXB_REQUIRE(a && a_scales && w && w_scales && y, "exb_fp8_matmul_fwd: null buffer");
    const int blocks = (K + kBlk - 1) / kBlk;
    EXB_REQUIRE(a_stride >= K && w_stride >= K && y_stride >= N, "exb_fp8_matmul_fwd: row strides smaller than the rows");
    EXB_REQUIRE(a_scale_stride >= M && w_scale_stride >= blocks, "exb_fp8_matmul_fwd: scale strides too small");
    EXB_REQUIRE(aligned16(a) && aligned16(w) && a_stride % 16 == 0 && w_stride % 16 == 0,
                "exb_fp8_matmul_fwd: the rows of a and w must start at multiples of 16 bytes");
    EXB_REQUIRE(rows::aligned_to(y, es) && rows::aligned_to(a_scales, 4) && rows::aligned_to(w_scales, 4) && rows::aligned_to(bias, 4),
                "exb_fp8_matmul_fwd: y, scales or bias not aligned to its element");
    if (M > 128) {
        PairParams p;
        if (int rc = encode(&p.tmA, a, M, K, a_stride, 128)) return rc;
        if (int rc = encode(&p.tmW, w, N, K, w_stride, 128)) return rc;
        p.a_scales = a_scales; p.w_scales = w_scales; p.bias = bias; p.y = y;
        p.a_scale_stride = a_scale_stride; p.w_scale_stride = w_scale_stride; p.y_stride = y_stride;
        p.M = (int)M; p.N = N; p.blocks = blocks; p.y_dtype = y_dtype;
        p.vec = rows::vector_rows(y, y_stride, es);
        p.m_tiles = (int)((M + kPairM - 1) / kPairM);
        p.n_tiles = (N + kPairN - 1) / kPairN;
        if ((int64_t)p.m_tiles * p.n_tiles > INT32_MAX / 2) return fail(EXB_ERR_UNSUPPORTED, "exb_fp8_matmul_fwd: %lld x %d is too large for one call", (long long)M, N);
        p.idesc = ptx::make_idesc(false, kPairM, kPairN);
        p.error = ctx->d_error;
        const int tiles = p.m_tiles * p.n_tiles, places = ctx->sm_count / 2;
        if (int rc = raise_smem_limit(ctx, fp8_matmul_pair_kernel)) return rc;
        return launch_pdl_cluster(ctx, "fp8_matmul_pair_kernel", fp8_matmul_pair_kernel, dim3(2 * (tiles < places ? tiles : places)), dim3(kPairThreads), dim3(2),
                                  (size_t)kPairStages * kPairStageBytes + kPairEpiWarps * kStageOut + 1024, static_cast<cudaStream_t>(stream), p);
    }
    MatmulParams p;
    if (int rc = encode(&p.tmA, a, M, K, a_stride, kTileM)) return rc;
    if (int rc = encode(&p.tmW, w, N, K, w_stride, kTileN)) return rc;
    p.a_scales = a_scales; p.w_scales = w_scales; p.bias = bias; p.y = y;
    p.a_scale_stride = a_scale_stride; p.w_scale_stride = w_scale_stride; p.y_stride = y_stride;
    p.M = (int)M; p.N = N; p.blocks = blocks; p.y_dtype = y_dtype;
    p.idesc = ptx::make_idesc(false, kTileM, kTileN);
    p.error = ctx->d_error;
    const int64_t gy = (M + kTileM - 1) / kTileM;
    if (gy > 65535) return fail(EXB_ERR_UNSUPPORTED, "exb_fp8_matmul_fwd: %lld rows are too many for one call", (long long)M);
    if (int rc = raise_smem_limit(ctx, fp8_matmul_kernel)) return rc;
    return launch_pdl(ctx, "fp8_matmul_kernel", fp8_matmul_kernel, dim3((N + kTileN - 1) / kTileN, (unsigned)gy), dim3(kThreads),
                      (size_t)kStages * kStageBytes + 1024, static_cast<cudaStream_t>(stream), p);
}
