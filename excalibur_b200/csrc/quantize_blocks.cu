// Rows of activations or weights -> 8-bit floating point (e4m3) with a scale for each block of 128 channels (of one row, or
// of 128 rows).  One pass over the input: a block's values stay in registers between its maximum and their conversion.
// Bound by memory: 2 (or 4) bytes in and 1 out for each element.  bf16, single rows: 8192 x 14336 in 56 us (6350 GB/s), 64 x 4096 in
// 1.7; rows of 14335, which are moved into place between lanes, 86 us.  Blocks of 128 rows: 4096 x 14336 in 29.8 us (5980 GB/s),
// rows of 14337 in 53.  fp32, 4096 x 14336: single rows 43.4 us (6770 GB/s), blocks of 128 rows 49.3 (5960 GB/s).
#include "rows_common.cuh"

namespace exb {
namespace {

using namespace rows;

constexpr int kThreads = 256;
constexpr int kRowsPerWarp = 4;                               // loads in flight per lane
constexpr int kTileRows = kThreads / 32 * kRowsPerWarp;       // a CTA's scales of a channel block fill a 128-byte line
constexpr int kShare = 2 * kBlock;

// Blocks of one row.  CTA: kTileRows rows x 256 channels, a warp kRowsPerWarp of the rows.
template <typename T, Layout kL>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T* __restrict__ x, int64_t x_stride, uint8_t* __restrict__ q,
                                                                 int64_t q_stride, float* __restrict__ scales, int64_t scale_stride,
                                                                 int64_t rows, int C, int shares, Span span) {
    pdl_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int share = blockIdx.x % shares, c0 = share * kShare, valid = C - c0;
    const int64_t r0 = (int64_t)(blockIdx.x / shares) * kTileRows + warp * kRowsPerWarp;
    const bool inside = r0 >= 8 && r0 + kRowsPerWarp <= rows - 8;
    Kept<T, kL> k[kRowsPerWarp];
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i)
        if (r0 + i < rows) k[i].load(x + (r0 + i) * x_stride + c0, valid, lane, span, inside);
    float m[kRowsPerWarp];
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
        if (r0 + i < rows) k[i].settle(x + (r0 + i) * x_stride + c0, valid, lane);
        else k[i].none();
        m[i] = k[i].amax();
    }
    quantize_shares<kRowsPerWarp>(
        [&](int i, float2(&v)[4]) { k[i].get(v); }, m, lane, scale_stride,
        [&](int i, int& n) {
            n = r0 + i < rows ? valid : 0;
            return q + (r0 + i) * q_stride + c0;
        },
        [&](int i) { return scales + 2 * share * scale_stride + r0 + i; });
}

// Blocks of 128 rows: a CTA has two neighbouring ones, its warps read shares of 256 channels of every 16th row.
constexpr int kTileWarps = 16, kTileSteps = kBlock / kTileWarps;

template <typename T, Layout kL>
__global__ void __launch_bounds__(kTileWarps * 32, sizeof(T) == 2 ? 2 : 1) quantize_tiles_kernel(const T* __restrict__ x, int64_t x_stride, uint8_t* __restrict__ q,
                                                                         int64_t q_stride, float* __restrict__ scales, int64_t scale_stride,
                                                                         int64_t rows, int C, int shares, Span span) {
    __shared__ float s_max[2][kTileWarps];
    pdl_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int share = blockIdx.x % shares, c0 = share * kShare, valid = C - c0;
    const int64_t rb = blockIdx.x / shares, r0 = rb * kBlock + warp;
    const bool inside = rb > 0 && (rb + 1) * kBlock <= rows - 8;
    Kept<T, kL> k[kTileSteps];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < kTileSteps; ++i) {
        const int64_t r = r0 + i * kTileWarps;
        if (r < rows) k[i].load(x + r * x_stride + c0, valid, lane, span, inside);
        else k[i].none();
    }
#pragma unroll
    for (int i = 0; i < kTileSteps; ++i) {
        k[i].settle(x + (r0 + i * kTileWarps) * x_stride + c0, valid, lane);
        m = fmaxf(m, k[i].amax());
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int half = lane >> 4;
    if ((lane & 15) == 0) s_max[half][warp] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTileWarps; ++i) m = fmaxf(m, s_max[half][i]);
    const float s = block_scale(m), inv = 1.f / s;
    if (warp == 0 && (lane & 15) == 0 && half * kBlock < valid) scales[rb * scale_stride + 2 * share + half] = s;
    if (lane * 8 >= valid) return;
#pragma unroll
    for (int i = 0; i < kTileSteps; ++i) {
        const int64_t r = r0 + i * kTileWarps;
        if (r >= rows) break;
        float2 v[4];
        k[i].get(v);
        store8_e4m3(q + r * q_stride + c0 + lane * 8, v, inv, valid - lane * 8);
    }
}

}  // namespace
}  // namespace exb

using namespace exb;

extern "C" int exb_quantize_blocks_fwd(exb_ctx* ctx, const exb_blocks_desc* d, const void* x, uint8_t* q, float* scales, void* stream) {
    EXB_REQUIRE(ctx != nullptr && d != nullptr, "exb_quantize_blocks_fwd: null context or descriptor");
    const int in_dtype = d->in_dtype, C = d->C, block_rows = d->block_rows;
    const int64_t n_rows = d->rows, x_stride = d->x_stride, q_stride = d->q_stride, scale_stride = d->scale_stride;
    const size_t es = rows::element_size(in_dtype);
    EXB_REQUIRE(es != 0, "exb_quantize_blocks_fwd: x must be EXB_F16, EXB_BF16 or EXB_F32, got %d", in_dtype);
    EXB_REQUIRE(n_rows >= 0 && C >= 1, "exb_quantize_blocks_fwd: bad shape (%lld rows of %d)", (long long)n_rows, C);
    EXB_REQUIRE(block_rows == 1 || block_rows == 128, "exb_quantize_blocks_fwd: blocks have 1 or 128 rows, got %d", block_rows);
    if (n_rows == 0) return EXB_OK;
    if (int rc = rows::check_device(ctx, "exb_quantize_blocks_fwd")) return rc;
    EXB_REQUIRE(x && q && scales, "exb_quantize_blocks_fwd: null buffer");
    const int64_t blocks = ((int64_t)C + rows::kBlock - 1) / rows::kBlock;
    EXB_REQUIRE(x_stride >= C && q_stride >= C, "exb_quantize_blocks_fwd: row strides smaller than the rows");
    EXB_REQUIRE(scale_stride >= (block_rows == 1 ? n_rows : blocks), "exb_quantize_blocks_fwd: scale stride %lld is too small", (long long)scale_stride);
    EXB_REQUIRE(rows::aligned_to(x, es) && rows::aligned_to(scales, 4), "exb_quantize_blocks_fwd: x or scales not aligned to its element");
    EXB_REQUIRE(aligned16(q) && q_stride % 16 == 0, "exb_quantize_blocks_fwd: q and its row stride must be multiples of 16 bytes");
    const rows::Place in[] = {rows::place_of(x, n_rows, C, x_stride, es)};
    const rows::Place out[] = {rows::place_of(q, n_rows, C, q_stride, 1),
                               block_rows == 1 ? rows::place_of(scales, blocks, n_rows, scale_stride, 4)
                                               : rows::place_of(scales, (n_rows - 1) / 128 + 1, blocks, scale_stride, 4)};
    EXB_REQUIRE(!rows::results_overlap(out, in), "exb_quantize_blocks_fwd: a result lies over x or over the other result");
    const int64_t shares = (blocks + 1) / 2;
    const int64_t grid = (block_rows == 1 ? (n_rows + kTileRows - 1) / kTileRows : (n_rows + 127) / 128) * shares;
    if (grid > INT32_MAX) return fail(EXB_ERR_UNSUPPORTED, "exb_quantize_blocks_fwd: %lld rows of %d are too many for one call", (long long)n_rows, C);
    const bool vec = C % 8 == 0 && rows::vector_rows(x, x_stride, es);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    rows::with_type(in_dtype, [&](auto t) {
        using T = decltype(t);
        const T* in = static_cast<const T*>(x);
        const rows::Span span = rows::span_of(x, n_rows, x_stride, C, es);
        if (block_rows == 1)
            launch_overlapped(ctx, vec ? quantize_rows_kernel<T, rows::kVectors> : quantize_rows_kernel<T, rows::kShifted>, dim3((unsigned)grid), dim3(kThreads), st, in, x_stride,
                              q, q_stride, scales, scale_stride, n_rows, C, (int)shares, span);
        else
            launch_overlapped(ctx, vec ? quantize_tiles_kernel<T, rows::kVectors> : quantize_tiles_kernel<T, rows::kShifted>, dim3((unsigned)grid), dim3(kTileWarps * 32), st, in,
                              x_stride, q, q_stride, scales, scale_stride, n_rows, C, (int)shares, span);
    });
    return after_launch("exb_quantize_blocks_fwd");
}
