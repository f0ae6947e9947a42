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
            if (!ptx::mbar_wait_bounded_warp(&tfull_bar[buf], (uint32_t)(b / 2) & 1u, &abort_flag, kMaxSpins)) {
                ok = false;
                break;
            }
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
