// Rows of activations or weights -> 8-bit floating point (e4m3) with a scale for each block of 128 channels (of one row, or
// of 128 rows).  One pass over the input: a block's values stay in registers between its maximum and their conversion.
// Bound by memory: 2 (or 4) bytes in and 1 out for each element.
#include "rows_common.cuh"

namespace exb {
namespace {

using namespace rows;

constexpr int kThreads = 256;
constexpr int kRowsPerWarp = 4;                               // loads in flight per lane
constexpr int kTileRows = kThreads / 32 * kRowsPerWarp;       // a CTA's scales of a channel block fill a 128-byte line
constexpr int kShare = 2 * kBlock;

// Blocks of one row.  CTA: kTileRows rows x 256 channels, a warp kRowsPerWarp of the rows.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T* __restrict__ x, int64_t x_stride, uint8_t* __restrict__ q,
                                                                 int64_t q_stride, float* __restrict__ scales, int64_t scale_stride,
                                                                 int64_t rows, int C, int shares) {
    pdl_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int share = blockIdx.x % shares, c0 = share * kShare, valid = C - c0;
    const int64_t r0 = (int64_t)(blockIdx.x / shares) * kTileRows + warp * kRowsPerWarp;
    float v[kRowsPerWarp][8];
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) load8<T, kVec>(x + (r0 + i) * x_stride + c0, r0 + i < rows ? valid : 0, lane, v[i]);
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i)
        quantize8<kVec>(v[i], r0 + i < rows ? valid : 0, lane, q + (r0 + i) * q_stride + c0, scales + 2 * share * scale_stride + r0 + i, scale_stride);
}

// Blocks of 128 rows: a CTA each.  A half-warp (kVec) or a warp reads a row's 128 channels.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) quantize_tiles_kernel(const T* __restrict__ x, int64_t x_stride, uint8_t* __restrict__ q,
                                                                  int64_t q_stride, float* __restrict__ scales, int64_t scale_stride,
                                                                  int64_t rows, int C, int blocks) {
    __shared__ float s_max[kThreads / 32];
    pdl_enter();
    constexpr int kLanes = kVec ? 16 : 32, kPer = kBlock / kLanes, kGroups = kThreads / kLanes, kSteps = kBlock / kGroups;
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    const int cb = blockIdx.x % blocks, c0 = cb * kBlock, valid = min(C - c0, kBlock);
    const int64_t rb = blockIdx.x / blocks, r0 = rb * kBlock + group;
    float v[kSteps][kPer], m = 0.f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int64_t r = r0 + i * kGroups;
        const T* at = x + r * x_stride + c0;
        if constexpr (kVec) {
            load8<T, true>(at, r < rows ? valid : 0, lane, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[i][j] = r < rows && j * 32 + lane < valid ? to_float<T>(at[j * 32 + lane]) : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int j = 0; j < kPer; ++j) m = fmaxf(m, fabsf(v[i][j]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) m = fmaxf(m, s_max[i]);
    const float s = block_scale(m), inv = 1.f / s;
    if (threadIdx.x == 0) scales[rb * scale_stride + cb] = s;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int64_t r = r0 + i * kGroups;
        if (r >= rows) break;
        uint8_t* at = q + r * q_stride + c0;
        if constexpr (kVec) {
            if (lane * 8 < valid) {
                const uint32_t lo = to_e4m3x2(v[i][0] * inv, v[i][1] * inv) | to_e4m3x2(v[i][2] * inv, v[i][3] * inv) << 16;
                const uint32_t hi = to_e4m3x2(v[i][4] * inv, v[i][5] * inv) | to_e4m3x2(v[i][6] * inv, v[i][7] * inv) << 16;
                *reinterpret_cast<uint2*>(at + lane * 8) = make_uint2(lo, hi);
            }
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                if (j * 32 + lane < valid) at[j * 32 + lane] = to_e4m3(v[i][j] * inv);
        }
    }
}

}  // namespace
}  // namespace exb

using namespace exb;

extern "C" int exb_quantize_blocks_fwd(exb_ctx* ctx, const void* x, int in_dtype, int64_t x_stride, uint8_t* q, int64_t q_stride,
                                       float* scales, int64_t scale_stride, int64_t n_rows, int C, int block_rows, void* stream) {
    EXB_REQUIRE(ctx != nullptr, "exb_quantize_blocks_fwd: null context");
    const size_t es = rows::element_size(in_dtype);
    EXB_REQUIRE(es != 0, "exb_quantize_blocks_fwd: x must be EXB_F16, EXB_BF16 or EXB_F32, got %d", in_dtype);
    EXB_REQUIRE(n_rows >= 0 && C >= 1, "exb_quantize_blocks_fwd: bad shape (%lld rows of %d)", (long long)n_rows, C);
    EXB_REQUIRE(block_rows == 1 || block_rows == 128, "exb_quantize_blocks_fwd: blocks have 1 or 128 rows, got %d", block_rows);
    if (n_rows == 0) return EXB_OK;
    EXB_REQUIRE(x && q && scales, "exb_quantize_blocks_fwd: null buffer");
    const int64_t blocks = ((int64_t)C + rows::kBlock - 1) / rows::kBlock;
    EXB_REQUIRE(x_stride >= C && q_stride >= C, "exb_quantize_blocks_fwd: row strides smaller than the rows");
    EXB_REQUIRE(scale_stride >= (block_rows == 1 ? n_rows : blocks), "exb_quantize_blocks_fwd: scale stride %lld is too small", (long long)scale_stride);
    EXB_REQUIRE(rows::aligned_to(x, es) && rows::aligned_to(scales, 4), "exb_quantize_blocks_fwd: x or scales not aligned to its element");
    EXB_REQUIRE(aligned16(q) && q_stride % 16 == 0, "exb_quantize_blocks_fwd: q and its row stride must be multiples of 16 bytes");
    const int64_t shares = (blocks + 1) / 2;
    const int64_t grid = block_rows == 1 ? (n_rows + kTileRows - 1) / kTileRows * shares : (n_rows + 127) / 128 * blocks;
    if (grid > INT32_MAX) return fail(EXB_ERR_UNSUPPORTED, "exb_quantize_blocks_fwd: %lld rows of %d are too many for one call", (long long)n_rows, C);
    const bool vec = C % 8 == 0 && rows::vector_rows(x, x_stride, es);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    rows::with_type(in_dtype, [&](auto t) {
        using T = decltype(t);
        const T* in = static_cast<const T*>(x);
        if (block_rows == 1)
            launch_overlapped(ctx, vec ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>, dim3((unsigned)grid), dim3(kThreads), st, in, x_stride,
                              q, q_stride, scales, scale_stride, n_rows, C, (int)shares);
        else
            launch_overlapped(ctx, vec ? quantize_tiles_kernel<T, true> : quantize_tiles_kernel<T, false>, dim3((unsigned)grid), dim3(kThreads), st, in, x_stride,
                              q, q_stride, scales, scale_stride, n_rows, C, (int)blocks);
    });
    return after_launch("exb_quantize_blocks_fwd");
}
