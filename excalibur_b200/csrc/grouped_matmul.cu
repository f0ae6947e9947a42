// Matrix products whose sums stay in TMEM over all of K: 8-bit integers with a scale for each row of a and each row of w, and products grouped
// by expert of 8-bit integers, fp16 or bf16:
//   y[m][n] = a_scales[m] * w_scales[e][n] * sum_k a[m][k] * w[e][n][k]  (+ bias[e][n]),   ends[e - 1] <= m < ends[e]
// (fp16 and bf16 without scales).  Sums of 8-bit integers are int32, exact; of fp16 and bf16 fp32.  An operand's rows are loaded in K blocks of
// 128 bytes, alike for all types, so the kernels differ in the kind of their MMAs and in what becomes of a sum.
#include "matmul_common.cuh"

#include <algorithm>
#include <type_traits>

namespace exb {
namespace {

using namespace product;

enum Kind { kInt8, kHalf, kBfloat };

struct ProductParams {
    CUtensorMap tmA, tmW;      // a: {bytes of K, rows}; w: {bytes of K, rows, experts}
    const float *a_scales, *w_scales, *bias;
    const int32_t* ends;
    void* y;
    int64_t y_stride;
    int M, N, blocks, experts, y_dtype, vec;      // experts 0: all rows are one's, and there are no ends
    int n_tiles, splits, stages;
    uint32_t idesc;
    int* error;
};

// ---- which rows are whose ------------------------------------------------------------------------
// Where each expert's rows end, and its tiles (kRows rows by one of n_tiles).  Ends come from the device and nobody has looked at them: one
// below those before it counts as theirs, one beyond the rows as their number, so that no row is two experts' and none is out of range.
// By all threads of a CTA; a barrier has to follow.
template <int kRows>
__device__ __forceinline__ void list_experts(const ProductParams& p, int2* table) {
    __shared__ int s_end[32], s_tiles[32];      // of each warp
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = (int)blockDim.x >> 5;
    int end = 0, tiles = 0;                      // of the experts before
    for (int e0 = 0; e0 < p.experts; e0 += (int)blockDim.x) {
        int v = e0 + tid < p.experts ? min(max(p.ends[e0 + tid], 0), p.M) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v = max(v, u);
        }
        __syncthreads();
        if (lane == 31) s_end[warp] = v;
        __syncthreads();
        int before = end;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) before = max(before, s_end[w]);
            end = max(end, s_end[w]);
        }
        v = max(v, before);
        const int begin = __shfl_up_sync(0xffffffffu, v, 1);
        int t = (v - (lane ? begin : before) + kRows - 1) / kRows * p.n_tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += u;
        }
        if (lane == 31) s_tiles[warp] = t;
        __syncthreads();
        t += tiles;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) t += s_tiles[w];
            tiles += s_tiles[w];
        }
        if (e0 + tid < p.experts) table[e0 + tid] = make_int2(v, t);
    }
}

// An expert's rows, and the number of a tile among its tiles.
struct Share {
    int expert, begin, end, tile;
};
template <int kRows>
__device__ __forceinline__ int all_tiles(const ProductParams& p, const int2* table) {
    return p.experts ? table[p.experts - 1].y : (p.M + kRows - 1) / kRows * p.n_tiles;
}
__device__ __forceinline__ Share share_of(const ProductParams& p, const int2* table, int tile) {
    if (!p.experts) return {0, 0, p.M, tile};
    int lo = 0, hi = p.experts - 1;      // the first with more tiles up to its end than that
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (table[mid].y > tile) hi = mid;
        else lo = mid + 1;
    }
    const int2 before = lo ? table[lo - 1] : make_int2(0, 0);
    return {lo, before.x, table[lo].x, tile - before.y};
}

template <Kind kKind>
__device__ __forceinline__ float sum_of(uint32_t raw) {
    return kKind == kInt8 ? (float)(int)raw : __uint_as_float(raw);
}

// ---- few rows of a group -------------------------------------------------------------------------
// Bound by the reading of w.  The roles of the operands are exchanged: w's rows are the MMA's 128 rows (lanes of TMEM), the rows of a its
// kCols columns, so that a narrow product wastes no tensor work and a thread has one channel of all rows.  With enough tiles for all
// SMs a CTA works on one after the other, the next one's loads under way while it stores (two accumulators in turn).  With fewer, the K blocks
// of a tile are divided over a cluster of up to 8 CTAs, so that enough of them ask for w at the same time; every CTA then
// finishes a share of the columns: the others send it their sums in one bulk copy each, counted by a barrier of its own.
// 8 bits: 16 x 128256 x 4096 takes 81.1 us (6490 GB/s), 16 x 65536 x 4096 43.3, 1 x 14336 x 4096 12.0 (4890 GB/s), 1 x 4096 x 4096 6.6: 3 to 4 us of start, exchange and
// end, and w at the copy rate between them.  2 x 4096 x 4096 fp16 of 2 of 8 experts 15.2 (w alone 10.2), 509 x 1500 x 2000 in 8 bits over 61 of 64 35.2 (28.3).
constexpr int kFewMostStages = 12;
constexpr int few_epi_warps(int cols) { return cols == 128 ? 16 : cols == 64 ? 8 : 4; }                   // up to 32 columns each
constexpr int few_stage_bytes(int cols) { return (128 + cols) * kBlk; }
// (columns that a CTA gets, of 16 by 7 CTAs: 3 from each of 6 others)
constexpr int few_received(int cols) { return cols == 16 ? 18 : cols; }
constexpr int few_smem(int cols, int stages, bool parts) { return stages * few_stage_bytes(cols) + (parts ? few_received(cols) * 512 : 0) + 1024; }

template <Kind kKind, int kCols>
__global__ void __launch_bounds__(96 + few_epi_warps(kCols) * 32, kCols == 128 ? 1 : 2) product_few_kernel(const __grid_constant__ ProductParams p) {
    constexpr int kStageBytes = few_stage_bytes(kCols), kEpi = few_epi_warps(kCols);
    const int stages = p.stages;
    constexpr int kMine = kCols * 4 / kEpi;      // columns of a warp
    constexpr int kTmem = 2 * kCols;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kFewMostStages], empty_bar[kFewMostStages], tfull_bar[2], tempty_bar[2], recv_bar;
    __shared__ uint32_t tmem_base_smem;
    __shared__ int abort_flag;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint32_t* part = reinterpret_cast<uint32_t*>(ring);                  // [column][128] behind the loop
    uint32_t* recv = part + stages * kStageBytes / 4;                    // [CTA, without this one][column of the share][128]
    int2* table = reinterpret_cast<int2*>(recv + (p.splits > 1 ? few_received(kCols) * 128 : 0));
    const int warp = ptx::uniform_warp(), lane = threadIdx.x & 31;
    const int rank = (int)blockIdx.x % p.splits, first = (int)blockIdx.x / p.splits, step = (int)gridDim.x / p.splits;
    const int b0 = (int)((int64_t)rank * p.blocks / p.splits), nb = (int)((int64_t)(rank + 1) * p.blocks / p.splits) - b0;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < stages; ++s) {
            ptx::mbar_init(&full_bar[s], 2);
            ptx::mbar_init(&empty_bar[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&tfull_bar[i], 1);
            ptx::mbar_init(&tempty_bar[i], kEpi);
        }
        ptx::mbar_init(&recv_bar, 1);
        ptx::fence_mbar_init();
        ptx::tma_prefetch_desc(&p.tmA);
        ptx::tma_prefetch_desc(&p.tmW);
    }
    __syncthreads();
    if (p.splits > 1) ptx::cluster_arrive();      // every CTA runs and its barriers are initialised: waited for before the first part is sent
    pdl_wait();
    if (p.experts) {
        list_experts<kCols>(p, table);
        __syncthreads();
    }
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
    const uint32_t ring0 = ptx::smem_u32(ring), full0 = ptx::smem_u32(full_bar), empty0 = ptx::smem_u32(empty_bar);
    const uint32_t tfull0 = ptx::smem_u32(tfull_bar), tempty0 = ptx::smem_u32(tempty_bar);
    const int total = all_tiles<kCols>(p, table);
    bool ok = true;
    auto tile_of = [&](int t, Share& s, int& m0, int& n0) {      // (an expert's tiles of the same rows of w follow one another)
        s = share_of(p, table, t);
        const int columns = (s.end - s.begin + kCols - 1) / kCols, n = s.tile / columns;
        m0 = s.begin + (s.tile - n * columns) * kCols;
        n0 = n * 128;
    };
    if (warp == 0 || warp == 2) {      // a loading warp for each operand
        const bool is_w = warp == 0;
        const uint32_t leader = ptx::elect_one() ? 1u : 0u;
        int s = 0;
        uint32_t phase = 1;      // (a fresh barrier's previous phase counts as complete)
        for (int t = first; t < total && ok; t += step) {
            Share of;
            int m0, n0;
            tile_of(t, of, m0, n0);
            for (int b = 0; b < nb; ++b) {
                if (!ptx::mbar_wait_quick_uniform(empty0 + s * 8, phase, &abort_flag, kMaxSpins)) {
                    ok = false;
                    break;
                }
                const uint32_t dst = ring0 + s * kStageBytes;
                if (is_w) {
                    ptx::mbar_arrive_expect_tx_u32(full0 + s * 8, 128 * kBlk, leader);
                    ptx::tma_load_3d_u32(dst, reinterpret_cast<uint64_t>(&p.tmW), full0 + s * 8, (b0 + b) * kBlk, n0, of.expert, leader);
                } else {
                    ptx::mbar_arrive_expect_tx_u32(full0 + s * 8, kCols * kBlk, leader);
                    ptx::tma_load_2d_u32(dst + 128 * kBlk, reinterpret_cast<uint64_t>(&p.tmA), full0 + s * 8, (b0 + b) * kBlk, m0, leader);
                }
                __syncwarp();      // (the elected lane may take a branch of its own; what follows is in registers of the whole warp)
                if (++s == stages) {
                    s = 0;
                    phase ^= 1u;
                }
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
        for (int t = first; t < total && ok; t += step) {
            if (!ptx::mbar_wait_quick_uniform(tempty0 + buf * 8, acc_phase, &abort_flag, kMaxSpins)) {
                ok = false;
                break;
            }
            ptx::tc_fence_after_sync();
            for (int b = 0; b < nb; ++b) {
                if (!ptx::mbar_wait_quick_uniform(full0 + s * 8, phase, &abort_flag, kMaxSpins)) {
                    ok = false;
                    break;
                }
                ptx::tc_fence_after_sync();
                const uint32_t w_lo = (uint32_t)d0 + ((uint32_t)(s * kStageBytes) >> 4), a_lo = w_lo + ((128 * kBlk) >> 4);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    ptx::tc_mma_lohi<kKind == kInt8>(tmem_base + buf * kCols, w_lo + 2 * ks, a_lo + 2 * ks, desc_hi, p.idesc, b | ks ? 1u : 0u, leader);
                ptx::tc_commit_u32(empty0 + s * 8, leader);
                __syncwarp();
                if (++s == stages) {
                    s = 0;
                    phase ^= 1u;
                }
            }
            if (!ok) break;
            ptx::tc_commit_u32(tfull0 + buf * 8, leader);
            __syncwarp();
            if (++buf == 2) {
                buf = 0;
                acc_phase ^= 1u;
            }
        }
        if (!ok) ptx::give_up(p.error, 2);
        __syncwarp();
    } else {
        const int q = warp & 3, c0 = ((warp - 3) >> 2) * kMine;
        int buf = 0;
        uint32_t acc_phase = 0;
        for (int t = first; t < total; t += step) {
            Share of;
            int m0, n0;
            tile_of(t, of, m0, n0);
            const int n = n0 + q * 32 + lane, rows = of.end - m0;
            // (asked for before there is anything to scale) this channel's scale and bias, and each row's scale in a lane of its own
            float ws = 1.f, as = 1.f, start = 0.f;
            if (p.splits == 1) {
                if (kKind == kInt8) {
                    ws = n < p.N ? p.w_scales[(int64_t)of.expert * p.N + n] : 0.f;
                    as = lane < kMine && c0 + lane < rows ? p.a_scales[m0 + c0 + lane] : 0.f;
                }
                if (p.bias && n < p.N) start = p.bias[(int64_t)of.expert * p.N + n];
            }
            if (!ptx::mbar_wait_quick_uniform(tfull0 + buf * 8, acc_phase, &abort_flag, kMaxSpins)) {
                ok = false;
                break;
            }
            __syncwarp();      // (what follows needs the warp together)
            ptx::tc_fence_after_sync();
            const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * kCols + c0);
            uint32_t raw[kMine / 16][16];
#pragma unroll
            for (int c = 0; c < kMine; c += 16) ptx::tmem_ld_32x32b_x16(taddr + c, raw[c / 16]);
#pragma unroll
            for (int c = 0; c < kMine; c += 16) ptx::tmem_ld_wait(raw[c / 16]);
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_u32(tempty0 + buf * 8);
            if (p.splits == 1) {
#pragma unroll
                for (int c = 0; c < kMine; ++c) {
                    if (c0 + c >= rows) break;
                    float v = sum_of<kKind>(raw[c / 16][c % 16]);
                    v = kKind == kInt8 ? fmaf(v, __shfl_sync(0xffffffffu, as, c % 32) * ws, start) : v + start;
                    if (n < p.N) store_one(p.y, p.y_dtype, (int64_t)(m0 + c0 + c) * p.y_stride + n, v);
                }
            } else {      // every MMA has read its operands: the sums take the ring's place
#pragma unroll
                for (int c = 0; c < kMine; ++c) part[(c0 + c) * 128 + q * 32 + lane] = raw[c / 16][c % 16];
            }
            if (++buf == 2) {
                buf = 0;
                acc_phase ^= 1u;
            }
        }
        if (!ok && lane == 0) atomicExch(p.error, 3);
    }
    if (p.splits > 1) {      // (a cluster has one tile at most)
        __syncwarp();
        ptx::cluster_wait();
        if (warp >= 3 && first < total) {
            Share of;
            int m0, n0;
            tile_of(first, of, m0, n0);
            // columns that this CTA finishes: [rank * share, rank * share + mine)
            const int cols = min(kCols, of.end - m0), share = (cols + p.splits - 1) / p.splits, mine = max(min(share, cols - rank * share), 0);
            const int et = (int)threadIdx.x - 96, row = (et & 31) * 4, n = n0 + row;      // a thread has four channels of a column
            if (et == 0) ptx::mbar_arrive_expect_tx(&recv_bar, (uint32_t)(mine * (p.splits - 1) * 512));
            if (ok) ptx::fence_proxy_async();
            asm volatile("bar.sync 1, %0;" ::"n"(kEpi * 32) : "memory");      // (all of them, whatever their waits gave)
            ok = ok && *static_cast<volatile int*>(&abort_flag) == 0;
            // lane r of the first warp sends CTA r its columns
            const int theirs = min(share, cols - lane * share);
            if (ok && warp == 3 && lane < p.splits && lane != rank && theirs > 0)
                ptx::copy_to_cta(ptx::map_to_cta(ptx::smem_u32(recv + (rank - (rank > lane)) * theirs * 128), (uint32_t)lane), ptx::smem_u32(part + lane * share * 128),
                                 (uint32_t)(theirs * 512), ptx::map_to_cta(ptx::smem_u32(&recv_bar), (uint32_t)lane));
            __syncwarp();
            float ws[4] = {1.f, 1.f, 1.f, 1.f}, start[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < p.N) {
                    if (kKind == kInt8) ws[j] = p.w_scales[(int64_t)of.expert * p.N + n + j];
                    if (p.bias) start[j] = p.bias[(int64_t)of.expert * p.N + n + j];
                }
            if (ok) ok = ptx::mbar_wait_quick_uniform(ptx::smem_u32(&recv_bar), 0, &abort_flag, kMaxSpins);
            if (!ok && lane == 0) atomicExch(p.error, 3);
            __syncwarp();
            ptx::cluster_arrive();      // no CTA leaves while parts may still be on their way to it or from it
            for (int c = et >> 5; ok && c < mine; c += kEpi) {
                const int m = m0 + rank * share + c;
                const float as = kKind == kInt8 ? p.a_scales[m] : 1.f;
                const uint32_t* own = part + (rank * share + c) * 128 + row;
                uint32_t sum[4];
#pragma unroll
                for (int s = 0; s < 8; ++s)
                    if (s < p.splits) {
                        const uint4 v = *reinterpret_cast<const uint4*>(s == rank ? own : recv + ((s - (s > rank)) * mine + c) * 128 + row);
                        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            sum[j] = !s ? u[j] : kKind == kInt8 ? sum[j] + u[j] : __float_as_uint(__uint_as_float(sum[j]) + __uint_as_float(u[j]));
                    }
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = kKind == kInt8 ? fmaf(sum_of<kKind>(sum[j]), as * ws[j], start[j]) : sum_of<kKind>(sum[j]) + start[j];
                store_four(p.y, p.y_dtype, p.y_stride, p.N, p.vec, m, n, v);
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
// Tiles of 256 rows of w by up to kWide rows of a by pairs of CTAs, persistent, with the operands' roles exchanged here too: the MMA's columns are as many as the
// tile has rows of a, in whole 32s, so that groups of any size cost the MMAs that they need (256 rows of a as the MMA's rows took 704 us for 8192 x 14336 x 4096 bf16
// over 8 experts, this takes 657); their loads are kWide / 2 rows of a for each CTA whatever the tile has.  An expert's rows are divided evenly between its tiles.  Each CTA keeps 128 rows of w and half of a's rows of a stage.
// TMEM holds two accumulators: the epilogue warps read one out, scale and store it while the MMAs fill the other.  A thread has a channel of all rows, and a
// warp stores 32 neighbours of a row at a time.
// 8 bits: 8192^3 takes 334 us from a cool GPU (3290 TOP/s; 390 when repeated for seconds, where the power limit sets the clock), 4096^3 49, of which the tensor pipe is
// active 64 %: 256 tiles for 74 pairs.  bf16, 8192 x 14336 x 4096 over 8 experts 657 to 693 (1390 to 1460 TFLOP/s).  Bound by the way from L2: 64 bytes a cycle and SM at 256
// columns, more with fewer.
constexpr int kPairEpiWarps = 8;                 // two per TMEM lane quarter, half of the accumulator's columns each
constexpr int pair_stage_bytes(int wide) { return (128 + wide / 2) * kBlk; }      // of one of the two CTAs
constexpr int pair_stages(int wide) { return wide == 256 ? 6 : 8; }
constexpr int pair_smem(int wide) { return pair_stages(wide) * pair_stage_bytes(wide) + 1024; }
constexpr int kPairThreads = 128 + kPairEpiWarps * 32;

// A thread's results of up to 32 rows from m on, in channel n.  (Neighbours put together in whole words took longer: 4048 x 7312 x 264 36.7 us, this way 29.0;
// so did whole vectors through shared memory, 34.8.)
template <typename T>
__device__ __forceinline__ void store_columns_as(const ProductParams& p, const float (&v)[32], int m, int n, int left) {
    T* y = static_cast<T*>(p.y) + (int64_t)m * p.y_stride + n;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        if (i < left && n < p.N) *y = rows::from_float<T>(v[i]);
        y += p.y_stride;
    }
}
__device__ __forceinline__ void store_columns(const ProductParams& p, const float (&v)[32], int m, int n, int left) {
    if (p.y_dtype == EXB_F16) store_columns_as<__half>(p, v, m, n, left);
    else if (p.y_dtype == EXB_BF16) store_columns_as<__nv_bfloat16>(p, v, m, n, left);
    else store_columns_as<float>(p, v, m, n, left);
}

template <Kind kKind, int kWide>
__global__ void __launch_bounds__(kPairThreads, 1) product_pair_kernel(const __grid_constant__ ProductParams p) {
    constexpr int kStages = pair_stages(kWide), kStageBytes = pair_stage_bytes(kWide);
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages], tfull_bar[2], tempty_bar[2];
    __shared__ uint32_t tmem_base_smem;
    __shared__ int abort_flag;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    int2* table = reinterpret_cast<int2*>(ring + kStages * kStageBytes);
    const int warp = ptx::uniform_warp(), lane = threadIdx.x & 31;
    const int rank = (int)__shfl_sync(0xffffffffu, ptx::cluster_ctarank(), 0);
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(&full_bar[s], 2);
            ptx::mbar_init(&empty_bar[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&tfull_bar[i], 1);
            ptx::mbar_init(&tempty_bar[i], 2 * kPairEpiWarps);
        }
        ptx::fence_mbar_init();
        ptx::tma_prefetch_desc(&p.tmA);
        ptx::tma_prefetch_desc(&p.tmW);
    }
    __syncwarp();
    pdl_wait();      // (before TMEM is taken: see kTmemOrder)
    if (p.experts) list_experts<kWide>(p, table);
    if (warp == 1) {
        ptx::tmem_alloc_pair(&tmem_base_smem, 2 * kWide);
        ptx::tmem_relinquish_pair();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();
    ptx::tc_fence_after_sync();
    pdl_launch_dependents();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_smem, 0);
    const uint32_t ring0 = ptx::smem_u32(ring), full0 = ptx::smem_u32(full_bar), empty0 = ptx::smem_u32(empty_bar);
    const uint32_t tfull0 = ptx::smem_u32(tfull_bar), tempty0 = ptx::smem_u32(tempty_bar);
    const int total = all_tiles<kWide>(p, table);
    // rows [m0, m0 + rows) of a, `wide` columns of the MMA; rows [n0, n0 + 256) of w
    struct Tile {
        int expert, m0, rows, wide, n0;
    };
    auto tile_of = [&](int t) {
        const Share s = share_of(p, table, t);
        const int all = s.end - s.begin, tiles = (all + kWide - 1) / kWide, each = ((all + tiles - 1) / tiles + 31) & ~31;
        int m, n;
        tile_at(s.tile, tiles, p.n_tiles, m, n);
        const int rows = min(each, all - m * each);
        return Tile{s.expert, s.begin + m * each, rows, (rows + 31) & ~31, n * 256};
    };
    if (warp == 0 || warp == 2) {      // a loading warp for each operand
        const bool is_w = warp == 0;
        const uint32_t leader = ptx::elect_one() ? 1u : 0u, counts = rank == 0 ? leader : 0u;
        const uint32_t full_lead = ptx::map_to_cta(full0, 0);
        bool ok = true;
        int s = 0;
        uint32_t phase = 1;      // (a fresh barrier's previous phase counts as complete)
        for (int t = first; t < total && ok; t += step) {
            const Tile of = tile_of(t);
            for (int b = 0; b < p.blocks; ++b) {
                if (!ptx::mbar_wait_quick_uniform(empty0 + s * 8, phase, &abort_flag, kMaxSpins)) {
                    ok = false;
                    break;
                }
                // (both CTAs' bytes are counted by rank 0)
                const uint32_t dst = ring0 + s * kStageBytes;
                if (is_w) {
                    ptx::mbar_arrive_expect_tx_u32(full0 + s * 8, 256 * kBlk, counts);
                    ptx::tma_load_3d_pair(dst, reinterpret_cast<uint64_t>(&p.tmW), full_lead + s * 8, b * kBlk, of.n0 + rank * 128, of.expert, leader);
                } else {
                    ptx::mbar_arrive_expect_tx_u32(full0 + s * 8, kWide * kBlk, counts);
                    ptx::tma_load_2d_pair(dst + 128 * kBlk, reinterpret_cast<uint64_t>(&p.tmA), full_lead + s * 8, b * kBlk, of.m0 + rank * (of.wide / 2), leader);
                }
                __syncwarp();      // (see the other kernel's)
                if (++s == kStages) {
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
            uint32_t phase = 0, acc_phase = 1;
            for (int t = first; t < total && ok; t += step) {
                const uint32_t idesc = p.idesc + ((uint32_t)(tile_of(t).wide >> 3) << 17);
                if (!ptx::mbar_wait_quick_uniform(tempty0 + buf * 8, acc_phase, &abort_flag, kMaxSpins)) {
                    ok = false;
                    break;
                }
                ptx::tc_fence_after_sync();
                for (int b = 0; b < p.blocks; ++b) {
                    if (!ptx::mbar_wait_quick_uniform(full0 + s * 8, phase, &abort_flag, kMaxSpins)) {
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after_sync();
                    const uint32_t w_lo = (uint32_t)d0 + ((uint32_t)(s * kStageBytes) >> 4), a_lo = w_lo + ((128 * kBlk) >> 4);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        ptx::tc_mma_lohi_pair<kKind == kInt8>(tmem_base + buf * kWide, w_lo + 2 * ks, a_lo + 2 * ks, desc_hi, idesc, b | ks ? 1u : 0u, leader);
                    ptx::tc_commit_pair_u32(empty0 + s * 8, leader);
                    __syncwarp();
                    if (++s == kStages) {
                        s = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                ptx::tc_commit_pair_u32(tfull0 + buf * 8, leader);
                __syncwarp();
                if (++buf == 2) {
                    buf = 0;
                    acc_phase ^= 1u;
                }
            }
            if (!ok) ptx::give_up(p.error, 2);
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int q = warp & 3, half = (warp >> 2) - 1;
        const uint32_t taddr0 = tmem_base + ((uint32_t)(q * 32) << 16);
        const uint32_t tempty_lead = ptx::map_to_cta(tempty0, 0);
        bool ok = true;
        int buf = 0;
        uint32_t acc_phase = 0;
        for (int t = first; t < total && ok; t += step) {
            const Tile of = tile_of(t);
            const int n = of.n0 + rank * 128 + q * 32 + lane, c0 = half * (of.wide / 2), c1 = min(c0 + of.wide / 2, of.rows);
            // (asked for before there is anything to scale) this channel's scale and bias, and each row's scale in a lane of its own
            const float ws = kKind == kInt8 && n < p.N ? p.w_scales[(int64_t)of.expert * p.N + n] : 0.f;
            const float start = p.bias && n < p.N ? p.bias[(int64_t)of.expert * p.N + n] : 0.f;
            float as[kWide / 64];
#pragma unroll
            for (int k = 0; k < kWide / 64; ++k) as[k] = kKind == kInt8 && c0 + k * 32 + lane < c1 ? p.a_scales[of.m0 + c0 + k * 32 + lane] : 0.f;
            if (!ptx::mbar_wait_bounded_uniform(tfull0 + buf * 8, acc_phase, &abort_flag, kMaxSpins)) {
                ok = false;
                break;
            }
            __syncwarp();      // (what follows needs the warp together)
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int k = 0; k < kWide / 64; ++k) {
                const int c = c0 + k * 32, rows = c1 - c;
                if (rows <= 0) break;
                uint32_t raw[2][16];
                const uint32_t taddr = taddr0 + (uint32_t)(buf * kWide + c);
                ptx::tmem_ld_32x32b_x16(taddr, raw[0]);
                if (rows > 16) ptx::tmem_ld_32x32b_x16(taddr + 16, raw[1]);
                ptx::tmem_ld_wait(raw[0]);
                ptx::tmem_ld_wait(raw[1]);
                if (rows <= 32) {
                    ptx::tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive_cluster_u32(tempty_lead + buf * 8);
                }
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float u = sum_of<kKind>(raw[i / 16][i % 16]);
                    v[i] = kKind == kInt8 ? fmaf(u, __shfl_sync(0xffffffffu, as[k], i) * ws, start) : u + start;
                }
                store_columns(p, v, of.m0 + c, n, rows);
            }
            if (c0 >= c1 && lane == 0) ptx::mbar_arrive_cluster_u32(tempty_lead + buf * 8);      // (none of its columns has a row)
            __syncwarp();
            if (++buf == 2) {
                buf = 0;
                acc_phase ^= 1u;
            }
        }
        if (!ok && lane == 0) atomicExch(p.error, 3);
    }
    __syncwarp();
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();      // neither CTA leaves while its peer may still signal its barriers or read its TMEM
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem_base, 2 * kWide);
    }
}

// Which kernel and how it divides the product.
//  - Up to 64 rows, or groups that have half as many on the average: the kernel for few rows, which has one tile for nearly every group.  But pairs load half as many
//    rows of a for each of w: with more than 24 rows, and tiles for three fifths of the pairs, they are the faster (K = 4096, us with few rows and in pairs: 17 x
//    14336 13.9 and 15.1, 32 x 14336 15.1 and 13.7, 64 x 11008 13.9 and 12.3, 64 x 128256 86.9 and 83.9, 64 x 4096 8.3 and 10.5; 400 x 1024 x 2048 int8 over 16
//    experts 13.3 and 11.5, 256 x 4096 x 4096 bf16 over 16 87 and 88).
//  - Otherwise the least of what was measured (8-bit and 16-bit alike: a K block has as many MMA cycles), us:
//    few rows, 128 columns: 5 + 2.2 where K is divided + 0.45 a block (128 x 4096 x 4096 11 to 12, in pairs 13);
//    pairs, 128 rows: 5 + 0.21 to 0.24 a block (512 x 4096 x 4096 11.8, 333 x 1000 x 1234 7.3);
//    pairs, 256 rows: 5 + 0.345 a block (512 x 4096 x 4096 16, 2048 x 4096 x 4096 26.9 and with 128 rows 32).
struct Plan {
    bool few;
    int tile, splits;      // rows of a in a tile, parts of K
    int each;              // CTAs of an SM (few)
};
Plan plan_for(int sms, int M, int N, int blocks, int experts) {
    const int64_t n_tiles = ((int64_t)N + 127) / 128, n_pairs = ((int64_t)N + 255) / 256;
    const int64_t groups = std::max(1, std::min(experts, M)), each = (M + groups - 1) / groups;
    auto m_tiles = [&](int rows) { return std::min<int64_t>(M, (M + groups * (rows - 1)) / rows); };                      // at most
    auto m_likely = [&](int rows) { return std::max<int64_t>(groups, (M + (groups > 1 ? groups * rows / 2 : rows - 1)) / rows); };
    // Parts of K, of at least two blocks each.  Clusters of several CTAs do not fill the SMs to the last: up to nine tenths are counted on.  Of one CTA an SM
    // as long as that leaves no more than three tenths of the SMs out; otherwise of two, and up to 1.65 an SM.  (64 rows, K = 4096, one and two CTAs an SM, each with
    // its best number of parts: N = 1024 and K = 14336 8.3 and 9.7 us, N = 4096 8.2 and 8.6, N = 6144 (32 rows) 9.2 and 8.1, N = 14336 15.0 and 15.8; 1 row, N = 4096
    // 6.5 and 6.4, N = 14336 12.3 and 13.4.)
    auto few = [&](int cols) -> Plan {
        const int64_t t = m_tiles(cols) * n_tiles;
        auto within = [&](int64_t places) { return std::max<int64_t>(1, std::min<int64_t>({8, places / t, blocks / 2})); };
        const int64_t one = t <= sms ? within(sms * 9 / 10) : 0;
        if (cols == 128) return {true, cols, (int)std::max<int64_t>(one, 1), 1};
        if (one && (t * one * 10 >= sms * 7 || one == 8)) return {true, cols, (int)one, 1};
        return {true, cols, (int)within(sms * 33 / 20), 2};
    };
    const int64_t rows = experts ? 2 * each : M;
    if (rows <= 64 && rows > 24 && m_likely(128) * n_pairs * 5 >= sms / 2 * 3) return {false, 128, 1, 1};
    if (rows <= 64) return few(rows <= 16 ? 16 : rows <= 32 ? 32 : 64);
    auto rounds = [](int64_t t, int64_t places) { return (double)((t + places - 1) / places); };
    const Plan narrow = few(128);
    const double few128 = 5.0 + (narrow.splits > 1 ? 2.2 : 0.0) + 0.45 * rounds(m_likely(128) * n_tiles * narrow.splits, sms) * ((blocks + narrow.splits - 1) / narrow.splits);
    const double rounds128 = rounds(m_likely(128) * n_pairs, sms / 2), pair128 = 5.0 + (rounds128 > 4 ? 0.235 : 0.212) * rounds128 * blocks;
    const double pair256 = 5.0 + 0.345 * rounds(m_likely(256) * n_pairs, sms / 2) * blocks;
    if (few128 < pair128 && few128 < pair256) return narrow;
    return {false, pair128 < pair256 ? 128 : 256, 1, 1};
}

// Rows of `bytes` of each expert in boxes of 128 bytes x box_rows, 128-byte swizzle; zeros beyond the matrix.
int encode_experts(const char* what, CUtensorMap* map, const void* base, int64_t rows, int64_t bytes, int64_t stride, int64_t experts, int64_t expert_stride,
                   int box_rows) {
    const auto fn = tensor_map_encoder();
    if (!fn) return fail(EXB_ERR_CUDA, "%s: the driver has no cuTensorMapEncodeTiled", what);
    cuuint64_t dims[3] = {(cuuint64_t)bytes, (cuuint64_t)rows, (cuuint64_t)experts}, strides[2] = {(cuuint64_t)stride, (cuuint64_t)expert_stride};
    cuuint32_t box[3] = {(cuuint32_t)kBlk, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(EXB_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
    return EXB_OK;
}

template <Kind kKind>
int run(exb_ctx* ctx, const char* what, ProductParams& p, const Plan& plan, const void* a, int64_t a_bytes, const void* w, int64_t K_bytes, int64_t w_bytes,
        int64_t expert_bytes, cudaStream_t st) {
    const int64_t M = p.M, experts = std::max(p.experts, 1), groups = std::min<int64_t>(experts, M);
    const size_t table = p.experts ? (size_t)p.experts * sizeof(int2) : 0;
    const int box_a = plan.few ? plan.tile : plan.tile / 2;
    if (int rc = encode_rows(what, &p.tmA, static_cast<const uint8_t*>(a), M, (int)K_bytes, a_bytes, box_a)) return rc;
    if (int rc = encode_experts(what, &p.tmW, w, p.N, K_bytes, w_bytes, experts, expert_bytes, 128)) return rc;
    const int rows = plan.tile, width = plan.few ? 128 : 256;
    p.n_tiles = (p.N + width - 1) / width;
    p.splits = plan.splits;
    const int64_t tiles = std::min<int64_t>(M, (M + groups * (rows - 1)) / rows) * p.n_tiles;      // at most
    if (tiles > INT32_MAX / 16) return fail(EXB_ERR_UNSUPPORTED, "%s: %lld x %d is too large for one call", what, (long long)M, p.N);
    // (pairs: the columns are the tile's)
    p.idesc = ptx::make_idesc(kKind == kInt8, plan.few ? 128 : 256, plan.few ? (uint32_t)plan.tile : 0u) | (kKind == kBfloat ? 1u << 7 | 1u << 10 : 0u);
    if (plan.few) {
        auto go = [&](auto c) {
            constexpr int kCols = decltype(c)::value;
            if (int rc = raise_smem_limit(ctx, product_few_kernel<kKind, kCols>)) return rc;
            const int64_t places = (int64_t)ctx->sm_count * plan.each;
            const int64_t grid = plan.splits > 1 ? tiles * plan.splits : std::min(tiles, places);
            // (more for one CTA an SM would keep the next kernel's from starting: 1 x 14336 x 4096 with 108, 150 and 220 KB 12.4, 12.0 and 12.5 us)
            const int room = (plan.each > 1 ? 108 : kCols == 128 ? 220 : 150) * 1024 - (int)table - few_smem(kCols, 0, plan.splits > 1);
            p.stages = std::min(kFewMostStages, room / few_stage_bytes(kCols));
            return launch_pdl_cluster(ctx, "product_few_kernel", product_few_kernel<kKind, kCols>, dim3((unsigned)grid), dim3(96 + few_epi_warps(kCols) * 32),
                                      dim3(plan.splits), (size_t)few_smem(kCols, p.stages, plan.splits > 1) + table, st, p);
        };
        if (plan.tile == 16) return go(std::integral_constant<int, 16>());
        if (plan.tile == 32) return go(std::integral_constant<int, 32>());
        if (plan.tile == 64) return go(std::integral_constant<int, 64>());
        return go(std::integral_constant<int, 128>());
    }
    const int64_t places = ctx->sm_count / 2;
    auto go = [&](auto c) {
        constexpr int kWide = decltype(c)::value;
        if (int rc = raise_smem_limit(ctx, product_pair_kernel<kKind, kWide>)) return rc;
        return launch_pdl_cluster(ctx, "product_pair_kernel", product_pair_kernel<kKind, kWide>, dim3((unsigned)(2 * std::min(tiles, places))), dim3(kPairThreads), dim3(2),
                                  (size_t)pair_smem(kWide) + table, st, p);
    };
    return plan.tile == 256 ? go(std::integral_constant<int, 256>()) : go(std::integral_constant<int, 128>());
}

constexpr int kMostExperts = 1024;
constexpr int kMostExactK = 131071;      // times 128^2: the largest sum of products below 2^31

int product_fwd(exb_ctx* ctx, const char* what, const exb_grouped_desc& d, bool grouped, const void* a, const float* a_scales, const void* w,
                const float* w_scales, const int32_t* ends, const float* bias, void* y, void* stream) {
    const int64_t M = d.M;
    const int N = d.N, K = d.K, experts = grouped ? d.experts : 1;
    const size_t es = d.dtype == EXB_I8 ? 1 : d.dtype == EXB_F16 || d.dtype == EXB_BF16 ? 2 : 0, ys = rows::element_size(d.y_dtype);
    EXB_REQUIRE(es != 0, "%s: a and w must be EXB_I8, EXB_F16 or EXB_BF16, got %d", what, d.dtype);
    EXB_REQUIRE(ys != 0, "%s: y must be EXB_F16, EXB_BF16 or EXB_F32, got %d", what, d.y_dtype);
    EXB_REQUIRE(M >= 0 && N >= 1 && K >= 1, "%s: bad shape (%lld x %d x %d)", what, (long long)M, N, K);
    EXB_REQUIRE(experts >= 1, "%s: %d experts", what, experts);
    if (experts > kMostExperts) return fail(EXB_ERR_UNSUPPORTED, "%s: at most %d experts, got %d", what, kMostExperts, experts);
    if (es == 1 && K > kMostExactK) return fail(EXB_ERR_UNSUPPORTED, "%s: int32 sums of 8-bit products hold K up to %d, got %d", what, kMostExactK, K);
    if (M > INT32_MAX - 256 || N > INT32_MAX - 256 || K > INT32_MAX / 2 - 256)
        return fail(EXB_ERR_UNSUPPORTED, "%s: %lld x %d x %d is too large for one call", what, (long long)M, N, K);
    if (M == 0) return EXB_OK;
    EXB_REQUIRE(a && w && y && (!grouped || ends), "%s: null buffer", what);
    EXB_REQUIRE((a_scales != nullptr) == (es == 1) && (w_scales != nullptr) == (es == 1), "%s: 8-bit integers have scales, other types none", what);
    EXB_REQUIRE(d.a_stride >= K && d.w_stride >= K && d.y_stride >= N, "%s: row strides smaller than the rows", what);
    const int64_t a_bytes = d.a_stride * (int64_t)es, w_bytes = d.w_stride * (int64_t)es;
    const int64_t expert_stride = experts > 1 ? d.expert_stride : (int64_t)N * d.w_stride, expert_bytes = expert_stride * (int64_t)es;
    EXB_REQUIRE(experts == 1 || expert_stride >= (N - 1) * d.w_stride + K, "%s: expert stride smaller than an expert", what);
    EXB_REQUIRE(aligned16(a) && aligned16(w) && a_bytes % 16 == 0 && w_bytes % 16 == 0 && expert_bytes % 16 == 0,
                "%s: the rows of a and w must start at multiples of 16 bytes", what);
    if (a_bytes >= 1ll << 40 || w_bytes >= 1ll << 40 || expert_bytes >= 1ll << 40) return fail(EXB_ERR_UNSUPPORTED, "%s: strides of 2^40 bytes or more", what);
    EXB_REQUIRE(rows::aligned_to(y, ys), "%s: y not aligned to its element", what);
    for (const void* q : {static_cast<const void*>(a_scales), static_cast<const void*>(w_scales), static_cast<const void*>(bias), static_cast<const void*>(ends)})
        EXB_REQUIRE(rows::aligned_to(q, 4), "%s: scales, bias or ends not aligned to their element", what);
    const int64_t w_span = (experts - 1) * expert_stride + (N - 1) * d.w_stride + K;      // (between its rows y may not lie either)
    const rows::Place in[] = {rows::place_of(a, M, K, d.a_stride, es),
                              experts == 1 ? rows::place_of(w, N, K, d.w_stride, es) : rows::place_of(w, 1, w_span, w_span, es),
                              rows::place_of(a_scales, 1, M, M, 4),
                              rows::place_of(w_scales, 1, (int64_t)experts * N, (int64_t)experts * N, 4),
                              rows::place_of(bias, 1, (int64_t)experts * N, (int64_t)experts * N, 4),
                              rows::place_of(grouped ? ends : nullptr, 1, experts, experts, 4)};
    const rows::Place out[] = {rows::place_of(y, M, N, d.y_stride, ys)};
    EXB_REQUIRE(!rows::results_overlap(out, in), "%s: y lies over an input", what);
    if (int rc = rows::check_device(ctx, what)) return rc;
    ProductParams p;
    p.a_scales = a_scales; p.w_scales = w_scales; p.bias = bias; p.ends = ends; p.y = y; p.y_stride = d.y_stride;
    p.M = (int)M; p.N = N; p.experts = grouped ? experts : 0; p.y_dtype = d.y_dtype;
    p.blocks = (int)(((int64_t)K * (int64_t)es + kBlk - 1) / kBlk);
    p.vec = rows::vector_rows(y, d.y_stride, ys);
    p.error = ctx->d_error;
    const Plan plan = plan_for(ctx->sm_count, p.M, N, p.blocks, p.experts);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t K_bytes = (int64_t)K * (int64_t)es;
    if (d.dtype == EXB_I8) return run<kInt8>(ctx, what, p, plan, a, a_bytes, w, K_bytes, w_bytes, expert_bytes, st);
    if (d.dtype == EXB_F16) return run<kHalf>(ctx, what, p, plan, a, a_bytes, w, K_bytes, w_bytes, expert_bytes, st);
    return run<kBfloat>(ctx, what, p, plan, a, a_bytes, w, K_bytes, w_bytes, expert_bytes, st);
}

}  // namespace
}  // namespace exb

using namespace exb;

extern "C" int exb_int8_matmul_fwd(exb_ctx* ctx, const exb_int8_desc* d, const int8_t* a, const float* a_scales, const int8_t* w, const float* w_scales,
                                   const float* bias, void* y, void* stream) {
    EXB_REQUIRE(ctx != nullptr && d != nullptr, "exb_int8_matmul_fwd: null context or descriptor");
    exb_grouped_desc g = {};
    g.M = d->M; g.N = d->N; g.K = d->K; g.dtype = EXB_I8; g.y_dtype = d->y_dtype; g.experts = 1;
    g.a_stride = d->a_stride; g.w_stride = d->w_stride; g.y_stride = d->y_stride;
    return product_fwd(ctx, "exb_int8_matmul_fwd", g, false, a, a_scales, w, w_scales, nullptr, bias, y, stream);
}

extern "C" int exb_grouped_matmul_fwd(exb_ctx* ctx, const exb_grouped_desc* d, const void* a, const float* a_scales, const void* w, const float* w_scales,
                                      const int32_t* ends, const float* bias, void* y, void* stream) {
    EXB_REQUIRE(ctx != nullptr && d != nullptr, "exb_grouped_matmul_fwd: null context or descriptor");
    return product_fwd(ctx, "exb_grouped_matmul_fwd", *d, true, a, a_scales, w, w_scales, ends, bias, y, stream);
}
