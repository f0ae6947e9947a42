// Matrix product in 8-bit floating point (e4m3 x e4m3) with an fp32 scale for each 128 of K and each row of a, and for each
// 128 x 128 of w:
//   y[m][n] = sum_b a_scales[b][m] * w_scales[n / 128][b] * sum_{k in b} a[m][k] * w[n][k]  (+ bias[n])
// The inner sums are tcgen05.mma into TMEM, a block of 128 at a time and two accumulators in turn; while the next block's
// MMAs run, the epilogue warps read the finished one back, scale it and add it to the sums that they hold in registers, in fp32.
#include "ptx_sm100.cuh"
#include "rows_common.cuh"
#include "tensor_map.cuh"

#include <algorithm>
#include <type_traits>

namespace exb {
namespace {

constexpr int kBlk = 128;                  // K block: bytes of a row in a stage, elements that share a scale
constexpr uint32_t kMaxSpins = 1u << 21;

// kTmemOrder: a kernel whose CTAs took TMEM while they wait for the previous kernel could take what CTAs of that one, started but not
// that far, still need, and both would wait for good.  So TMEM is taken behind griddepcontrol.wait, and the next kernel is let in
// (griddepcontrol.launch_dependents) only behind that.
struct MatmulParams {
    CUtensorMap tmA, tmW;
    const float *a_scales, *w_scales, *bias;
    void* y;
    int64_t a_scale_stride, w_scale_stride, y_stride;
    int M, N, blocks, y_dtype, vec;
    int m_tiles, n_tiles, splits;
    uint32_t idesc;
    int* error;
};

__device__ __forceinline__ void store_one(void* y, int dtype, int64_t at, float v) {
    if (dtype == EXB_F16) static_cast<__half*>(y)[at] = __float2half_rn(v);
    else if (dtype == EXB_BF16) static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
    else static_cast<float*>(y)[at] = v;
}

// Four neighbouring channels of a row.
__device__ __forceinline__ void store_four(const MatmulParams& p, int m, int n, const float (&v)[4]) {
    const int64_t at = (int64_t)m * p.y_stride + n;
    if (p.vec && n + 4 <= p.N) {
        if (p.y_dtype == EXB_F32)
            *reinterpret_cast<float4*>(static_cast<float*>(p.y) + at) = make_float4(v[0], v[1], v[2], v[3]);
        else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + at) =
                p.y_dtype == EXB_F16 ? make_uint2(rows::float_to_pair(v[0], v[1], __half()), rows::float_to_pair(v[2], v[3], __half()))
                                     : make_uint2(rows::float_to_pair(v[0], v[1], __nv_bfloat16()), rows::float_to_pair(v[2], v[3], __nv_bfloat16()));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < p.N) store_one(p.y, p.y_dtype, at + j, v[j]);
    }
}

// ---- few rows of a -----------------------------------------------------------------------------
// Bound by the reading of w.  The roles of the operands are exchanged: w's rows are the MMA's 128 rows (lanes of TMEM), the rows of a its
// kCols columns, so that a narrow product wastes no tensor work and a thread has one channel of all rows.  The K blocks of a
// tile are divided over a cluster of up to 8 CTAs, so that enough of them ask for w at the same time.  Every CTA then finishes a
// share of the columns: the others send it their parts in one bulk copy each, counted by a barrier of its own, and it sums them in
// the order of the CTAs.  (Read out of the others' shared memory between cluster barriers the exchange took 3600 cycles for 16
// columns and 8000 for 64.)
// 1 x 4096 x 4096 takes 6.0 us, 1 x 14336 x 4096 12.4 (4730 GB/s), 64 x 14336 x 4096 16.4 (3710 GB/s): about 3 us of start, exchange and
// end, and w at 5 TB/s or so between them.  Without w's latency to hide (131 x 2432 x 9088, 16.6) the 0.42 us of a K block are what counts.
constexpr int kFewBufs = 4;          // accumulators in turn: TMEM has room
constexpr int kFewTable = 16;        // blocks whose scales are in shared memory at a time
constexpr int few_stages(int cols) { return cols == 128 ? 4 : cols == 64 ? 3 : cols == 32 ? 4 : 5; }      // (two CTAs fit an SM up to 64 columns)
constexpr int few_epi_warps(int cols) { return cols == 128 ? 16 : cols == 64 ? 8 : 4; }
constexpr int few_stage_bytes(int cols) { return (128 + cols) * kBlk; }
// (columns that a CTA gets, of 16 by 7 CTAs: 3 from each of 6 others)
constexpr int few_received(int cols) { return cols == 16 ? 18 : cols; }
constexpr int few_smem(int cols) { return few_stages(cols) * few_stage_bytes(cols) + kFewTable * cols * 4 + few_received(cols) * 512 + 1024; }

template <int kCols>
__global__ void __launch_bounds__(96 + few_epi_warps(kCols) * 32, kCols == 128 ? 1 : 2) fp8_matmul_few_kernel(const __grid_constant__ MatmulParams p) {
    constexpr int kStages = few_stages(kCols), kStageBytes = few_stage_bytes(kCols), kEpi = few_epi_warps(kCols);
    constexpr int kMine = kCols * 4 / kEpi;      // columns of a warp
    constexpr int kTmem = kFewBufs * kCols;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages], tfull_bar[kFewBufs], tempty_bar[kFewBufs], recv_bar;
    __shared__ uint32_t tmem_base_smem;
    __shared__ int abort_flag;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* table = reinterpret_cast<float*>(ring + kStages * kStageBytes);      // [block][column]: a's scale x w's
    float* recv = table + kFewTable * kCols;                                    // [CTA, without this one][column of the share][128]
    float* part = reinterpret_cast<float*>(ring);                               // [column][128] behind the loop
    const int warp = ptx::uniform_warp(), lane = threadIdx.x & 31;
    const int rank = (int)blockIdx.x % p.splits, n0 = (int)blockIdx.x / p.splits * 128, m0 = blockIdx.y * kCols;
    const int b0 = (int)((int64_t)rank * p.blocks / p.splits), nb = (int)((int64_t)(rank + 1) * p.blocks / p.splits) - b0;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(&full_bar[s], 1);
            ptx::mbar_init(&empty_bar[s], 1);
        }
        for (int i = 0; i < kFewBufs; ++i) {
            ptx::mbar_init(&tfull_bar[i], 1);
            ptx::mbar_init(&tempty_bar[i], kEpi);
        }
        ptx::mbar_init(&recv_bar, 1);
        ptx::fence_mbar_init();
        ptx::tma_prefetch_desc(&p.tmA);
        ptx::tma_prefetch_desc(&p.tmW);
    }
    __syncthreads();
    const uint32_t ring0 = ptx::smem_u32(ring), full0 = ptx::smem_u32(full_bar), empty0 = ptx::smem_u32(empty_bar);
    const uint32_t tfull0 = ptx::smem_u32(tfull_bar), tempty0 = ptx::smem_u32(tempty_bar);
    // columns that this CTA finishes: [rank * share, rank * share + mine)
    const int cols = min(kCols, p.M - m0), share = (cols + p.splits - 1) / p.splits, mine = max(min(share, cols - rank * share), 0);
    if (p.splits > 1) {      // every CTA runs and its barriers are initialised: waited for before the first part is sent
        ptx::cluster_arrive();
        if (threadIdx.x == 0) ptx::mbar_arrive_expect_tx(&recv_bar, (uint32_t)(mine * (p.splits - 1) * 512));
        __syncwarp();
    }
    float acc[kMine];
    bool ok = true;
    pdl_wait();
    // TMEM is taken when the previous kernel is done, and the next one may start when it is taken (see kTmemOrder).  The loads do not wait
    // for it.
    uint32_t tmem_base = 0;
    if (warp != 0 && warp != 2) {
        if (warp == 1) {
            ptx::tmem_alloc(&tmem_base_smem, kTmem);
            ptx::tmem_relinquish();
            ptx::tc_fence_before_sync();
        }
        asm volatile("bar.sync 2, %0;" ::"n"(kEpi * 32 + 32) : "memory");
        ptx::tc_fence_after_sync();
        tmem_base = __shfl_sync(0xffffffffu, tmem_base_smem, 0);
        pdl_launch_dependents();
    }
    if (warp == 0 || warp == 2) {      // a loading warp for each operand
        const bool is_w = warp == 0;
        const uint32_t leader = ptx::elect_one() ? 1u : 0u;
        const uint64_t map = is_w ? reinterpret_cast<uint64_t>(&p.tmW) : reinterpret_cast<uint64_t>(&p.tmA);
        const uint32_t dst = ring0 + (is_w ? 0 : 128 * kBlk);
        const int row0 = is_w ? n0 : m0;
        int s = 0;
        uint32_t phase = 1;      // (a fresh barrier's previous phase counts as complete)
        for (int b = 0; b < nb; ++b) {
            if (b >= kStages && !ptx::mbar_wait_quick_uniform(empty0 + s * 8, phase, &abort_flag, kMaxSpins)) {
                ok = false;
                break;
            }
            ptx::mbar_arrive_expect_tx_u32(full0 + s * 8, kStageBytes, is_w ? leader : 0u);
            ptx::tma_load_2d_u32(dst + s * kStageBytes, map, full0 + s * 8, (b0 + b) * kBlk, row0, leader);
            __syncwarp();      // (the elected lane may take a branch of its own; what follows is in registers of the whole warp)
            if (++s == kStages) {
                s = 0;
                phase ^= 1u;
            }
        }
        if (!ok && lane == 0) ptx::give_up(p.error, 1);
        __syncwarp();
    } else if (warp == 1) {
        const uint32_t leader = ptx::elect_one() ? 1u : 0u;
        const uint64_t d0 = ptx::make_smem_desc(ring0, kBlk);
        const uint32_t desc_hi = (uint32_t)(d0 >> 32);
        int s = 0, buf = 0;
        uint32_t phase = 0, acc_phase = 1;
        for (int b = 0; b < nb; ++b) {
            if (!ptx::mbar_wait_quick_uniform(full0 + s * 8, phase, &abort_flag, kMaxSpins) ||
                !ptx::mbar_wait_quick_uniform(tempty0 + buf * 8, acc_phase, &abort_flag, kMaxSpins)) {
                ok = false;
                break;
            }
            ptx::tc_fence_after_sync();
            const uint32_t w_lo = (uint32_t)d0 + ((uint32_t)(s * kStageBytes) >> 4), a_lo = w_lo + ((128 * kBlk) >> 4);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
                ptx::tc_mma_f8<false>(tmem_base + buf * kCols, w_lo + 2 * ks, a_lo + 2 * ks, desc_hi, p.idesc, ks ? 1u : 0u, leader);
            if (b + kStages < nb) ptx::tc_commit_u32(empty0 + s * 8, leader);
            ptx::tc_commit_u32(tfull0 + buf * 8, leader);
            __syncwarp();
            if (++s == kStages) {
                s = 0;
                phase ^= 1u;
            }
            if (++buf == kFewBufs) {
                buf = 0;
                acc_phase ^= 1u;
            }
        }
        if (!ok) ptx::give_up(p.error, 2);
        __syncwarp();
    } else {
        const int q = warp & 3, c0 = ((warp - 3) >> 2) * kMine, et = (int)threadIdx.x - 96;
        const float* sw = p.w_scales + (int64_t)(n0 / kBlk) * p.w_scale_stride + b0;
        const int n = n0 + q * 32 + lane;
        const float start = p.bias && rank == 0 && n < p.N ? __ldg(p.bias + n) : 0.f;      // (asked for before there is anything to add)
#pragma unroll
        for (int i = 0; i < kMine; ++i) acc[i] = start;
        int buf = 0;
        uint32_t acc_phase = 0;
        for (int b = 0; b < nb; ++b) {
            if (b % kFewTable == 0) {
                if (b) asm volatile("bar.sync 1, %0;" ::"n"(kEpi * 32) : "memory");
                // a thread has one column; eight loads at a time are under way
                constexpr int kStep = kEpi * 32 / kCols;
                const int rows = min(nb - b, kFewTable), c = et % kCols;
                const float* sa = p.a_scales + (int64_t)(b0 + b) * p.a_scale_stride + m0 + c;
                for (int k = et / kCols; k < rows; k += 8 * kStep) {
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        v[j] = c < cols && k + j * kStep < rows ? __ldg(sa + (int64_t)(k + j * kStep) * p.a_scale_stride) * __ldg(sw + b + k + j * kStep) : 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (k + j * kStep < rows) table[(k + j * kStep) * kCols + c] = v[j];
                }
                asm volatile("bar.sync 1, %0;" ::"n"(kEpi * 32) : "memory");
            }
            // a warp that has given up still meets the others at their barrier
            if (ok && !ptx::mbar_wait_quick_uniform(tfull0 + buf * 8, acc_phase, &abort_flag, kMaxSpins)) ok = false;
            if (!ok) continue;
            __syncwarp();      // (what follows needs the warp together)
            ptx::tc_fence_after_sync();
            const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * kCols + c0);
            const float4* s4 = reinterpret_cast<const float4*>(table + (b % kFewTable) * kCols + c0);
#pragma unroll
            for (int c = 0; c < kMine; c += 16) {
                uint32_t raw[16];
                ptx::tmem_ld_32x32b_x16(taddr + c, raw);
                float4 s[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] = s4[c / 4 + j];
                ptx::tmem_ld_wait(raw);
                if (c + 16 == kMine) {
                    ptx::tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive_u32(tempty0 + buf * 8);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    acc[c + 4 * j] = fmaf(__uint_as_float(raw[4 * j]), s[j].x, acc[c + 4 * j]);
                    acc[c + 4 * j + 1] = fmaf(__uint_as_float(raw[4 * j + 1]), s[j].y, acc[c + 4 * j + 1]);
                    acc[c + 4 * j + 2] = fmaf(__uint_as_float(raw[4 * j + 2]), s[j].z, acc[c + 4 * j + 2]);
                    acc[c + 4 * j + 3] = fmaf(__uint_as_float(raw[4 * j + 3]), s[j].w, acc[c + 4 * j + 3]);
                }
            }
            if (++buf == kFewBufs) {
                buf = 0;
                acc_phase ^= 1u;
            }
        }
        if (!ok && lane == 0) atomicExch(p.error, 3);
        if (p.splits == 1) {
            if (ok && n < p.N) {
#pragma unroll
                for (int i = 0; i < kMine; ++i)
                    if (m0 + c0 + i < p.M) store_one(p.y, p.y_dtype, (int64_t)(m0 + c0 + i) * p.y_stride + n, acc[i]);
            }
        } else if (ok) {      // every MMA has read its operands: the parts take the ring's place
#pragma unroll
            for (int i = 0; i < kMine; ++i) part[(c0 + i) * 128 + q * 32 + lane] = acc[i];
        }
    }
    if (p.splits > 1) {
        __syncwarp();
        ptx::cluster_wait();
        if (warp >= 3) {
            const int et = (int)threadIdx.x - 96, row = (et & 31) * 4;      // a thread has four channels of a column
            if (ok) ptx::fence_proxy_async();
            asm volatile("bar.sync 1, %0;" ::"n"(kEpi * 32) : "memory");      // (all of them, whatever their waits gave)
            ok = ok && *static_cast<volatile int*>(&abort_flag) == 0;
            // lane r of the first warp sends CTA r its columns
            const int theirs = min(share, cols - lane * share);
            if (ok && warp == 3 && lane < p.splits && lane != rank && theirs > 0)
                ptx::copy_to_cta(ptx::map_to_cta(ptx::smem_u32(recv + (rank - (rank > lane)) * theirs * 128), (uint32_t)lane), ptx::smem_u32(part + lane * share * 128),
                                 (uint32_t)(theirs * 512), ptx::map_to_cta(ptx::smem_u32(&recv_bar), (uint32_t)lane));
            __syncwarp();
            if (ok) ok = ptx::mbar_wait_quick_uniform(ptx::smem_u32(&recv_bar), 0, &abort_flag, kMaxSpins);
            if (!ok && lane == 0) atomicExch(p.error, 3);
            __syncwarp();
            ptx::cluster_arrive();      // no CTA leaves while parts may still be on their way to it or from it
            for (int c = et >> 5; ok && c < mine; c += kEpi) {
                const float* own = part + (rank * share + c) * 128 + row;
                float sum[4];
#pragma unroll
                for (int s = 0; s < 8; ++s)
                    if (s < p.splits) {
                        const float4 v = *reinterpret_cast<const float4*>(s == rank ? own : recv + ((s - (s > rank)) * mine + c) * 128 + row);
                        sum[0] = s ? sum[0] + v.x : v.x;
                        sum[1] = s ? sum[1] + v.y : v.y;
                        sum[2] = s ? sum[2] + v.z : v.z;
                        sum[3] = s ? sum[3] + v.w : v.w;
                    }
                store_four(p, m0 + rank * share + c, n0 + row, sum);
            }
        } else {
            ptx::cluster_arrive();
        }
        __syncwarp();
        ptx::cluster_wait();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, kTmem);
    }
}

// ---- CTA pairs ---------------------------------------------------------------------------------
// Tiles of 256 x 256 by pairs of CTAs, persistent.  Each CTA keeps 128 rows of a and half of w's rows of a stage, 32 KB for
// 512 cycles of MMA: 64 bytes per cycle and SM from L2 (a lone CTA's tile of 128 x 128 needs 128).  TMEM holds two accumulators of
// 256 columns; a thread's sums are 128 registers.  8192^3 takes 441 to 458 us (2400 to 2490 TFLOP/s) from a cool GPU and 543 (2020
// TFLOP/s) when repeated for seconds, where the power limit sets the clock; 4096^3 67.  Bound by the epilogue: a block's read out of
// TMEM and its multiply-adds take 800 cycles, the MMAs 512 of these (the tensor pipe is active 59 % of 4096^3).  K is not divided
// between pairs: clusters of two pairs took 131 x 2432 x 9088 in 18.8 us where the kernel above takes 16.6, and 1695 x 3315 x 9300,
// which leaves most of a second wave empty, in 92 instead of 70 (a CTA's start costs more than the wave).
constexpr int kPairM = 256;
constexpr int kPairEpiWarps = 8;                 // two per TMEM lane quarter, half of the accumulator's columns each
constexpr int pair_stage_bytes(int n) { return (kPairM + n) / 2 * kBlk; }      // of one of the two CTAs
constexpr int pair_stages(int n) { return n == 256 ? 6 : 8; }

// Results of 32 rows x up to 128 bytes per warp, in units of 16 bytes that are XOR-ed with the row: a thread writes its row's units
// and the warp reads whole rows, both without bank conflicts.
constexpr int kStageOut = 32 * 128;

// Columns [col, col + 2 * kPairs) of 32 rows from row0 on: sums in `acc` (a thread has a row), through shared memory to y in whole vectors.
template <typename T, int kPairs>
__device__ __forceinline__ void store_rows(const float2 (&acc)[kPairs], uint8_t* stage, T* y, int64_t y_stride, int row0, int col, int M, int N, bool vec,
                                           int lane) {
    constexpr int kPer = 16 / (int)sizeof(T);                                                   // columns in a unit,
    constexpr int kUnits = 2 * kPairs / kPer < 8 ? 2 * kPairs / kPer : 8, kCols = kUnits * kPer;      // units and columns in a pass
    constexpr int kRows = 32 / kUnits;                                                          // rows that the warp writes at a time
    const int sub = lane / kUnits, u = lane % kUnits;
    auto unit = [&](int r, int i) { return reinterpret_cast<uint4*>(stage + r * 128 + ((i ^ (r & 7)) << 4)); };
    auto element = [&](int r, int e) { return reinterpret_cast<const T*>(unit(r, e / kPer))[e % kPer]; };
#pragma unroll
    for (int c0 = 0; c0 < 2 * kPairs; c0 += kCols) {
        if (col + c0 >= N) break;
        const int left = N - col - c0;
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const float2* v = acc + (c0 + i * kPer) / 2;
            if constexpr (sizeof(T) == 4)
                *unit(lane, i) = make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
            else
                *unit(lane, i) = make_uint4(rows::float_to_pair(v[0].x, v[0].y, T()), rows::float_to_pair(v[1].x, v[1].y, T()),
                                            rows::float_to_pair(v[2].x, v[2].y, T()), rows::float_to_pair(v[3].x, v[3].y, T()));
        }
        __syncwarp();
        T* out = y + (int64_t)row0 * y_stride + col + c0;
        if (left < kCols) {
            for (int r = 0; r < 32 && row0 + r < M; ++r) {
#pragma unroll
                for (int c = lane; c < kCols; c += 32)
                    if (c < left) out[r * y_stride + c] = element(r, c);
            }
        } else if (vec) {
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int r = i * kRows + sub;
                if (row0 + r < M) *reinterpret_cast<uint4*>(out + r * y_stride + u * kPer) = *unit(r, u);
            }
        } else {
            // Rows that start anywhere: kUnits - 1 vectors at multiples of 16 bytes, put together of two units each, and 16 bytes before
            // and behind them element by element.  (fp16, 4048 x 7313 x 264 takes
            // 42.9 us, element by element 51.8, and 4048 x 7312 x 264 29: sectors that two passes write a part of each are the difference.)
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int r = i * kRows + sub;
                if (row0 + r >= M) continue;
                T* to = out + r * y_stride;
                const int o = (int)((16 - (reinterpret_cast<uintptr_t>(to) & 15)) & 15);      // bytes before the first multiple of 16
                if (o == 0) {
                    *reinterpret_cast<uint4*>(to + u * kPer) = *unit(r, u);
                    continue;
                }
                if (u < kUnits - 1) {
                    const uint4 a = *unit(r, u), b = *unit(r, u + 1);
                    uint32_t x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                    if (o & 8) {
#pragma unroll
                        for (int k = 0; k < 6; ++k) x[k] = x[k + 2];
                    }
                    if (o & 4) {
#pragma unroll
                        for (int k = 0; k < 5; ++k) x[k] = x[k + 1];
                    }
                    const int sh = (o & 2) * 8;
                    *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(to) + o + u * 16) =
                        make_uint4(__funnelshift_r(x[0], x[1], sh), __funnelshift_r(x[1], x[2], sh), __funnelshift_r(x[2], x[3], sh), __funnelshift_r(x[3], x[4], sh));
                }
#pragma unroll
                for (int k = 0; k < kPer; k += kUnits)      // as many elements before the first vector and behind the last as a unit has
                    if (k + u < kPer) {
                        const int e = (k + u) * (int)sizeof(T) < o ? k + u : kCols - kPer + k + u;
                        to[e] = element(r, e);
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

// Warps 0 and 2 load, warp 1 issues the MMAs, two warpgroups keep the sums: 2 x 224 + 56 registers (2 x 176 + 152 with
// 128 columns) are the 3 x 168 of the launch.
constexpr int kPairThreads = 128 + kPairEpiWarps * 32;
template <int kRegs> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }

template <int kPairN>
__global__ void __launch_bounds__(kPairThreads, 1) fp8_matmul_pair_kernel(const __grid_constant__ MatmulParams p) {
    constexpr int kPairStages = pair_stages(kPairN), kPairStageBytes = pair_stage_bytes(kPairN), kPairCols = kPairN / 2, kBufs = 512 / kPairN;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kPairStages], empty_bar[kPairStages], tfull_bar[kBufs];
    __shared__ uint32_t tmem_base_smem;
    __shared__ int abort_flag;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = ptx::uniform_warp(), lane = threadIdx.x & 31;
    const int rank = (int)__shfl_sync(0xffffffffu, ptx::cluster_ctarank(), 0);
    const int total = p.m_tiles * p.n_tiles, first = blockIdx.x >> 1, step = gridDim.x >> 1;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < kPairStages; ++s) {
            ptx::mbar_init(&full_bar[s], 1 + 2 * kPairEpiWarps);
            ptx::mbar_init(&empty_bar[s], 1);
        }
        for (int i = 0; i < kBufs; ++i) ptx::mbar_init(&tfull_bar[i], 1);
        ptx::fence_mbar_init();
        ptx::tma_prefetch_desc(&p.tmA);
        ptx::tma_prefetch_desc(&p.tmW);
    }
    pdl_wait();      // (before TMEM is taken: see kTmemOrder)
    if (warp == 1) {
        ptx::tmem_alloc_pair(&tmem_base_smem, 512);
        ptx::tmem_relinquish_pair();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();
    ptx::tc_fence_after_sync();
    pdl_launch_dependents();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_smem, 0);
    const uint32_t ring0 = ptx::smem_u32(ring), full0 = ptx::smem_u32(full_bar), empty0 = ptx::smem_u32(empty_bar);
    const uint32_t tfull0 = ptx::smem_u32(tfull_bar), full_lead = ptx::map_to_cta(full0, 0);
    if (warp < 4) {
        fewer_registers<kPairN == 256 ? 56 : 152>();
        // The MMAs of a block take 512 (256 columns) or 256 cycles, a wait for a barrier that is complete 90, a load 120 and more.  So
        // the operands have a loading warp each (with one for both, its 560 cycles a block were what the kernel waited for), and the
        // issuing warp has one wait per block: the epilogue warps' arrival that frees the accumulator of block g is counted by the
        // barrier of the stage that block g + kBufs is loaded into.  (Lanes that look at a barrier each are no way out: one look at
        // 12 barriers took 280 cycles.)
        if (warp == 0 || warp == 2) {
            const bool is_w = warp == 2;
            const uint32_t leader = ptx::elect_one() ? 1u : 0u, counts = rank == 0 && !is_w ? leader : 0u;
            const uint64_t map = is_w ? reinterpret_cast<uint64_t>(&p.tmW) : reinterpret_cast<uint64_t>(&p.tmA);
            const uint32_t dst = ring0 + (is_w ? 128 * kBlk : 0);
            bool ok = true;
            int s = 0;
            uint32_t phase = 1;      // (a fresh barrier's previous phase counts as complete)
            for (int t = first; t < total && ok; t += step) {
                int mt, nt;
                tile_at(t, p.m_tiles, p.n_tiles, mt, nt);
                const int row0 = is_w ? nt * kPairN + rank * (kPairN / 2) : mt * kPairM + rank * 128;
                for (int b = 0; b < p.blocks; ++b) {
                    if (!ptx::mbar_wait_quick_uniform(empty0 + s * 8, phase, &abort_flag, kMaxSpins)) {
                        ok = false;
                        break;
                    }
                    // (both CTAs' bytes are counted by rank 0)
                    ptx::mbar_arrive_expect_tx_u32(full0 + s * 8, 2 * kPairStageBytes, counts);
                    ptx::tma_load_2d_pair(dst + s * kPairStageBytes, map, full_lead + s * 8, b * kBlk, row0, leader);
                    __syncwarp();      // (see the other kernel's)
                    if (++s == kPairStages) {
                        s = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (!ok && lane == 0) ptx::give_up(p.error, 1);
            __syncwarp();
        } else if (warp == 1) {
            if (rank == 0) {      // issues for both
                const uint32_t leader = ptx::elect_one() ? 1u : 0u;
                const uint64_t d0 = ptx::make_smem_desc(ring0, kBlk);
                const uint32_t desc_hi = (uint32_t)(d0 >> 32);
                bool ok = true;
                int s = 0, buf = 0;
                uint32_t phase = 0;
                for (int t = first; t < total && ok; t += step) {
                    for (int b = 0; b < p.blocks; ++b) {
                        if (!ptx::mbar_wait_quick_uniform(full0 + s * 8, phase, &abort_flag, kMaxSpins)) {
                            ok = false;
                            break;
                        }
                        ptx::tc_fence_after_sync();
                        const uint32_t a_lo = (uint32_t)d0 + ((uint32_t)(s * kPairStageBytes) >> 4), w_lo = a_lo + ((128 * kBlk) >> 4);
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            ptx::tc_mma_f8<true>(tmem_base + buf * kPairN, a_lo + 2 * ks, w_lo + 2 * ks, desc_hi, p.idesc, ks ? 1u : 0u, leader);
                        ptx::tc_commit_pair_u32(tfull0 + buf * 8, leader);
                        ptx::tc_commit_pair_u32(empty0 + s * 8, leader);
                        __syncwarp();
                        if (++s == kPairStages) {
                            s = 0;
                            phase ^= 1u;
                        }
                        if (++buf == kBufs) buf = 0;
                    }
                }
                if (!ok) ptx::give_up(p.error, 2);
            }
            __syncwarp();
        }
    } else {
        more_registers<kPairN == 256 ? 224 : 176>();
        const int q = warp & 3, part = (warp >> 2) - 1;
        uint8_t* stage = ring + kPairStages * kPairStageBytes + (warp - 4) * kStageOut;
        const uint32_t taddr0 = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(part * kPairCols);
        bool ok = true;
        int buf = 0, next = kBufs;      // accumulator, and the stage of the block that takes it next
        uint32_t acc_phase = 0;
        if (lane < kBufs) ptx::mbar_arrive_cluster_u32(full_lead + lane * 8);      // all accumulators are free
        __syncwarp();
        for (int t = first; t < total && ok; t += step) {
            int mt, nt;
            tile_at(t, p.m_tiles, p.n_tiles, mt, nt);
            const int row = mt * kPairM + rank * 128 + q * 32 + lane, col = nt * kPairN + part * kPairCols;
            // This row's and these columns' scales: two blocks' are on their way, each in registers of its own (a register that is
            // moved has to be there first, and the loop would wait for memory in every block).
            const float* sa = p.a_scales + (row < p.M ? row : 0);
            const float* sw = p.w_scales + (int64_t)(col < p.N ? col / kBlk : 0) * p.w_scale_stride;
            float a_scale[2] = {__ldg(sa), 0.f}, w_scale[2] = {__ldg(sw), 0.f};
            if (p.blocks > 1) {
                a_scale[1] = __ldg(sa += p.a_scale_stride);
                w_scale[1] = __ldg(++sw);
            }
            float2 acc[kPairCols / 2];
#pragma unroll
            for (int i = 0; i < kPairCols / 2; ++i) acc[i] = make_float2(0.f, 0.f);
            if (p.bias) {      // (while the first block is on its way)
#pragma unroll
                for (int i = 0; i < kPairCols / 2; ++i) {
                    if (col + 2 * i < p.N) acc[i].x = __ldg(p.bias + col + 2 * i);
                    if (col + 2 * i + 1 < p.N) acc[i].y = __ldg(p.bias + col + 2 * i + 1);
                }
            }
            for (int b = 0; b < p.blocks && ok; b += 2) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (b + k >= p.blocks) break;
                    const float s = a_scale[k] * w_scale[k];
                    if (b + k + 2 < p.blocks) {
                        a_scale[k] = __ldg(sa += p.a_scale_stride);
                        w_scale[k] = __ldg(++sw);
                    }
                    if (!ptx::mbar_wait_quick_uniform(tfull0 + buf * 8, acc_phase, &abort_flag, kMaxSpins)) {
                        ok = false;
                        break;
                    }
                    __syncwarp();      // (what follows needs the warp together)
                    ptx::tc_fence_after_sync();
                    const uint32_t taddr = taddr0 + (uint32_t)(buf * kPairN);
#pragma unroll
                    for (int c = 0; c < kPairCols; c += 16) {
                        uint32_t raw[16];
                        ptx::tmem_ld_32x32b_x16(taddr + c, raw);
                        ptx::tmem_ld_wait(raw);
                        if (c + 16 == kPairCols) {
                            ptx::tc_fence_before_sync();
                            __syncwarp();
                            if (lane == 0) ptx::mbar_arrive_cluster_u32(full_lead + next * 8);
                        }
                        // (two sums at an instruction save power, 1 % of 8192^3 under the cap; with 128 columns, where the loop's length
                        // counts, one at a time is faster: 512 x 4096 x 4096 14.9 us, 16.6 in twos)
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float u = __uint_as_float(raw[2 * j]), v = __uint_as_float(raw[2 * j + 1]);
                            float2& to = acc[c / 2 + j];
                            if constexpr (kPairN == 256) to = __ffma2_rn(make_float2(u, v), make_float2(s, s), to);
                            else to = make_float2(fmaf(u, s, to.x), fmaf(v, s, to.y));
                        }
                    }
                    if (++next == kPairStages) next = 0;
                    if (++buf == kBufs) {
                        buf = 0;
                        acc_phase ^= 1u;
                    }
                }
            }
            if (!ok) break;
            const int row0 = row - lane;
            if (p.y_dtype == EXB_F16) store_rows(acc, stage, static_cast<__half*>(p.y), p.y_stride, row0, col, p.M, p.N, p.vec, lane);
            else if (p.y_dtype == EXB_BF16) store_rows(acc, stage, static_cast<__nv_bfloat16*>(p.y), p.y_stride, row0, col, p.M, p.N, p.vec, lane);
            else store_rows(acc, stage, static_cast<float*>(p.y), p.y_stride, row0, col, p.M, p.N, p.vec, lane);
        }
        if (!ok && lane == 0) atomicExch(p.error, 3);
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();      // neither CTA leaves while its peer may still signal its barriers or read its TMEM
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem_base, 512);
    }
}

// Which kernel and how it divides the product: the one whose time is least by what was measured of each (graph-captured calls, us):
//  - few rows, up to 64 columns: the only one that does not compute rows that are not there;
//  - few rows, 128 columns: 5 + 2.2 where K is divided + 0.42 for each K block that a CTA works on one after the other
//    (131 x 2432 x 9088 in one part 34.4, in two 20.8, in three 16.6; 512 x 1024 x 8192 in four 13.4);
//  - pairs with tiles of 128 columns: 4.5 + 0.335 a block (512 x 4096 x 4096 14.9, in 256 columns 18.1);
//  - pairs with tiles of 256 columns: 5 + 0.43 a block (256 x 14336 x 4096 19.9, in 128 columns 25.5; 4096^3 67 and 81).
struct Plan {
    bool few;
    int tile, splits;      // columns of a tile
};
Plan plan_for(int sms, int M, int N, int blocks) {
    const int64_t n_tiles = ((int64_t)N + 127) / 128;
    // Parts of K, of at least two blocks each.  Clusters of several CTAs do not fill the SMs to the last: up to nine tenths are counted on.
    // Up to 64 columns an SM has room for two CTAs; they are only used, and up to 1.65 an SM, where one each would leave a fifth
    // of the SMs out (1 row, K = 4096, N = 4096 in 4 parts 6.0, in 8 6.7; N = 6144 in 3 parts 7.6, in 5 7.4, in 6 10.4; 64 rows, N = 4096 8.7 and
    // 9.7, N = 6144 12.3, 10.6 and 15.7).
    auto parts = [&](int64_t tiles, bool two) {
        auto within = [&](int64_t places) { return std::max<int64_t>(1, std::min<int64_t>({8, places / tiles, blocks / 2})); };
        const int64_t s = within(sms * 9 / 10);
        return (int)(two && tiles * s * 5 < sms * 4 ? within(sms * 33 / 20) : s);
    };
    if (M <= 64) return {true, M <= 16 ? 16 : M <= 32 ? 32 : 64, parts(n_tiles, true)};
    auto rounds = [](int64_t tiles, int64_t places) { return (double)((tiles + places - 1) / places); };
    const int64_t few_tiles = ((int64_t)M + 127) / 128 * n_tiles, m_pairs = ((int64_t)M + kPairM - 1) / kPairM;
    const int splits = parts(few_tiles, false);
    const double few = 5.0 + (splits > 1 ? 2.2 : 0.0) + 0.42 * rounds(few_tiles * splits, sms) * ((blocks + splits - 1) / splits);
    const double pair128 = 4.5 + 0.335 * rounds(m_pairs * n_tiles, sms / 2) * blocks;
    const double pair256 = 5.0 + 0.43 * rounds(m_pairs * (((int64_t)N + 255) / 256), sms / 2) * blocks;
    if (few < pair128 && few < pair256 && few_tiles / n_tiles <= 65535) return {true, 128, splits};
    return {false, pair128 < pair256 ? 128 : 256, 1};
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

extern "C" int exb_fp8_matmul_fwd(exb_ctx* ctx, const exb_matmul_desc* d, const uint8_t* a, const float* a_scales, const uint8_t* w,
                                  const float* w_scales, const float* bias, void* y, void* stream) {
    EXB_REQUIRE(ctx != nullptr && d != nullptr, "exb_fp8_matmul_fwd: null context or descriptor");
    const int64_t M = d->M, a_stride = d->a_stride, a_scale_stride = d->a_scale_stride, w_stride = d->w_stride, w_scale_stride = d->w_scale_stride,
                  y_stride = d->y_stride;
    const int N = d->N, K = d->K, y_dtype = d->y_dtype;
    const size_t es = rows::element_size(y_dtype);
    EXB_REQUIRE(es != 0, "exb_fp8_matmul_fwd: y must be EXB_F16, EXB_BF16 or EXB_F32, got %d", y_dtype);
    EXB_REQUIRE(M >= 0 && N >= 1 && K >= 1, "exb_fp8_matmul_fwd: bad shape (%lld x %d x %d)", (long long)M, N, K);
    if (M > INT32_MAX - 256 || N > INT32_MAX - 256 || K > INT32_MAX - 256)
        return fail(EXB_ERR_UNSUPPORTED, "exb_fp8_matmul_fwd: %lld x %d x %d is too large for one call", (long long)M, N, K);
    if (M == 0) return EXB_OK;
    if (int rc = rows::check_device(ctx, "exb_fp8_matmul_fwd")) return rc;
    EXB_REQUIRE(a && a_scales && w && w_scales && y, "exb_fp8_matmul_fwd: null buffer");
    const int blocks = (K + kBlk - 1) / kBlk;
    EXB_REQUIRE(a_stride >= K && w_stride >= K && y_stride >= N, "exb_fp8_matmul_fwd: row strides smaller than the rows");
    EXB_REQUIRE(a_scale_stride >= M && w_scale_stride >= blocks, "exb_fp8_matmul_fwd: scale strides too small");
    EXB_REQUIRE(aligned16(a) && aligned16(w) && a_stride % 16 == 0 && w_stride % 16 == 0,
                "exb_fp8_matmul_fwd: the rows of a and w must start at multiples of 16 bytes");
    EXB_REQUIRE(rows::aligned_to(y, es) && rows::aligned_to(a_scales, 4) && rows::aligned_to(w_scales, 4) && rows::aligned_to(bias, 4),
                "exb_fp8_matmul_fwd: y, scales or bias not aligned to its element");
    const rows::Place in[] = {rows::place_of(a, M, K, a_stride, 1), rows::place_of(a_scales, blocks, M, a_scale_stride, 4), rows::place_of(w, N, K, w_stride, 1),
                              rows::place_of(w_scales, (N - 1) / kBlk + 1, blocks, w_scale_stride, 4), rows::place_of(bias, 1, N, N, 4)};
    const rows::Place out[] = {rows::place_of(y, M, N, y_stride, es)};
    EXB_REQUIRE(!rows::results_overlap(out, in), "exb_fp8_matmul_fwd: y lies over an input");
    MatmulParams p;
    p.a_scales = a_scales; p.w_scales = w_scales; p.bias = bias; p.y = y;
    p.a_scale_stride = a_scale_stride; p.w_scale_stride = w_scale_stride; p.y_stride = y_stride;
    p.M = (int)M; p.N = N; p.blocks = blocks; p.y_dtype = y_dtype;
    p.vec = rows::vector_rows(y, y_stride, es);
    p.error = ctx->d_error;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const Plan plan = plan_for(ctx->sm_count, (int)M, N, blocks);
    if ((int64_t)((M + 127) / 128) * ((N + 127) / 128) > INT32_MAX / 16)
        return fail(EXB_ERR_UNSUPPORTED, "exb_fp8_matmul_fwd: %lld x %d is too large for one call", (long long)M, N);
    if (plan.few) {
        const int cols = plan.tile;
        p.m_tiles = (int)((M + cols - 1) / cols);
        p.n_tiles = (N + 127) / 128;
        p.splits = plan.splits;
        if (int rc = encode(&p.tmA, a, M, K, a_stride, cols)) return rc;
        if (int rc = encode(&p.tmW, w, N, K, w_stride, 128)) return rc;
        p.idesc = ptx::make_idesc(false, 128, (uint32_t)cols);
        auto go = [&](auto c) {
            constexpr int kCols = decltype(c)::value;
            if (int rc = raise_smem_limit(ctx, fp8_matmul_few_kernel<kCols>)) return rc;
            return launch_pdl_cluster(ctx, "fp8_matmul_few_kernel", fp8_matmul_few_kernel<kCols>, dim3((unsigned)p.n_tiles * p.splits, (unsigned)p.m_tiles),
                                      dim3(96 + few_epi_warps(kCols) * 32), dim3(p.splits), (size_t)few_smem(kCols), st, p);
        };
        if (cols == 16) return go(std::integral_constant<int, 16>());
        if (cols == 32) return go(std::integral_constant<int, 32>());
        if (cols == 64) return go(std::integral_constant<int, 64>());
        return go(std::integral_constant<int, 128>());
    }
    if (int rc = encode(&p.tmA, a, M, K, a_stride, 128)) return rc;
    const int wide = plan.tile;
    if (int rc = encode(&p.tmW, w, N, K, w_stride, wide / 2)) return rc;
    p.m_tiles = (int)((M + kPairM - 1) / kPairM);
    p.n_tiles = (N + wide - 1) / wide;
    p.splits = 1;
    p.idesc = ptx::make_idesc(false, kPairM, (uint32_t)wide);
    const int tiles = p.m_tiles * p.n_tiles, places = ctx->sm_count / 2;
    auto go = [&](auto c) {
        constexpr int kN = decltype(c)::value;
        if (int rc = raise_smem_limit(ctx, fp8_matmul_pair_kernel<kN>)) return rc;
        return launch_pdl_cluster(ctx, "fp8_matmul_pair_kernel", fp8_matmul_pair_kernel<kN>, dim3(2 * (tiles < places ? tiles : places)), dim3(kPairThreads), dim3(2),
                                  (size_t)pair_stages(kN) * pair_stage_bytes(kN) + kPairEpiWarps * kStageOut + 1024, st, p);
    };
    return wide == 256 ? go(std::integral_constant<int, 256>()) : go(std::integral_constant<int, 128>());
}
