// Rows of activations or weights -> 8-bit integers with a scale for each row: q = the whole number nearest to x / scale.
// One pass: a row's elements stay in registers, packed, between its largest magnitude and their conversion.  A magnitude's bits order as whole numbers, so
// the largest costs one instruction for two 16-bit elements, and an infinity or a NaN comes out on top.  x * r + 1.5 * 2^23 is rounded once, at
// the whole numbers: its low byte is q, exactly the nearest to x * r, ties to the even one.
// Bound by memory: 2 (or 4) bytes in and 1 out for each element.  8192 x 14336 bf16 takes 53.6 us (6570 GB/s), 8192 x 8192 fp16 33.0 (6100), 65536 x 256 10.5 (4790),
// 1 x 4096 1.2; rows of 4095, which are moved into place between lanes, 27.1 instead of 17.2 for 8192 of 4096; rows of 65536, read twice, 68 for 1024.
#include "rows_common.cuh"

namespace exb {
namespace {

using namespace rows;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kShare = 256;      // elements of a warp's share
constexpr float kMagic = 12582912.f;

// The bits of a lane's largest magnitude, as fp32.
template <typename T, Layout kL>
__device__ __forceinline__ uint32_t largest_bits(const Kept<T, kL>& k) {
    uint32_t m = 0;
    if constexpr (Kept<T, kL>::kPacked) {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __vmaxu2(m, k.w[i] & 0x7fff7fffu);
        const uint32_t one = max(m & 0xffffu, m >> 16);
        return __float_as_uint(pair_to_float(one, T()).x);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, k.w[i] & 0x7fffffffu);
        return m;
    }
}

struct Scale {
    float scale, inverse;      // inverse 0: a row without a scale
};
__device__ __forceinline__ Scale scale_of(uint32_t bits) {
    if (bits >= 0x7f800000u) return {NAN, 0.f};
    const float s = fmaxf(__uint_as_float(bits) / 127.f, kSmallestScale);
    return {s, 1.f / s};
}

// A lane's 8 neighbours, of which `valid` are the row's.
template <typename T, Layout kL>
__device__ __forceinline__ void store_share(const Kept<T, kL>& k, int8_t* q, float inverse, int valid) {
    float2 v[4];
    k.get(v);
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = __ffma2_rn(v[i], make_float2(inverse, inverse), make_float2(kMagic, kMagic));
        b[i] = __byte_perm(__float_as_uint(v[i].x), __float_as_uint(v[i].y), 0x0040);
    }
    uint2 o = make_uint2(__byte_perm(b[0], b[1], 0x5410), __byte_perm(b[2], b[3], 0x5410));
    if (inverse == 0.f) o = make_uint2(0, 0);
    if (valid >= 8) {
        *reinterpret_cast<uint2*>(q) = o;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < valid) q[j] = (int8_t)((j < 4 ? o.x : o.y) >> (8 * (j & 3)));
    }
}

// kRowWarps warps of a CTA have kRows rows, up to kShares shares of each (every kRowWarps-th).
template <typename T, Layout kL, int kRowWarps, int kShares, int kRows>
__global__ void __launch_bounds__(kRowWarps > kWarps ? kRowWarps * 32 : kThreads)
quantize_whole_rows_kernel(const T* __restrict__ x, int64_t x_stride, int8_t* __restrict__ q, int64_t q_stride, float* __restrict__ scales, int64_t rows, int C,
                           Span span) {
    static_assert(kRowWarps == 1 || kRows == 1, "several rows for a warp alone");
    constexpr int kGroups = kRowWarps > kWarps ? 1 : kWarps / kRowWarps;      // of warps with rows of their own
    __shared__ uint32_t s_max[kGroups * kRowWarps];
    pdl_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % kRowWarps;
    const int64_t r0 = ((int64_t)blockIdx.x * kGroups + warp / kRowWarps) * kRows;
    const bool inside = r0 >= 8 && r0 + kRows <= rows - 8;
    Kept<T, kL> k[kRows][kShares];
    auto valid = [&](int r, int i) { return r0 + r < rows ? C - (i * kRowWarps + part) * kShare : 0; };      // elements of the share
    auto at = [&](int r, int i) { return x + (r0 + r) * x_stride + (i * kRowWarps + part) * kShare; };
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int i = 0; i < kShares; ++i) {
            if (valid(r, i) > 0) k[r][i].load(at(r, i), valid(r, i), lane, span, inside);
            else k[r][i].none();
        }
    uint32_t m[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        m[r] = 0;
#pragma unroll
        for (int i = 0; i < kShares; ++i) {
            if (valid(r, i) > 0) k[r][i].settle(at(r, i), valid(r, i), lane);
            m[r] = max(m[r], largest_bits(k[r][i]));
        }
        m[r] = __reduce_max_sync(0xffffffffu, m[r]);
    }
    if constexpr (kRowWarps > 1) {
        if (lane == 0) s_max[warp] = m[0];
        __syncthreads();
        const int first = warp / kRowWarps * kRowWarps;
#pragma unroll
        for (int i = 0; i < kRowWarps; ++i) m[0] = max(m[0], s_max[first + i]);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (r0 + r >= rows) break;
        const Scale s = scale_of(m[r]);
        if (part == 0 && lane == 0) scales[r0 + r] = s.scale;
#pragma unroll
        for (int i = 0; i < kShares; ++i)
            if (lane * 8 < valid(r, i)) store_share(k[r][i], q + (r0 + r) * q_stride + (i * kRowWarps + part) * kShare + lane * 8, s.inverse, valid(r, i) - lane * 8);
    }
}

// Rows that no CTA's registers hold: read twice, the second time mostly out of L2.
template <typename T, Layout kL>
__global__ void __launch_bounds__(kThreads) quantize_long_rows_kernel(const T* __restrict__ x, int64_t x_stride, int8_t* __restrict__ q, int64_t q_stride,
                                                                      float* __restrict__ scales, int64_t rows, int C, Span span) {
    __shared__ uint32_t s_max[kWarps];
    pdl_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = blockIdx.x;
    const bool inside = r >= 8 && r < rows - 8;
    const T* at = x + r * x_stride;
    Kept<T, kL> k;
    uint32_t m = 0;
    for (int c0 = warp * kShare; c0 < C; c0 += kThreads * 8) {
        k.load(at + c0, C - c0, lane, span, inside);
        k.settle(at + c0, C - c0, lane);
        m = max(m, largest_bits(k));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) s_max[warp] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) m = max(m, s_max[i]);
    const Scale s = scale_of(m);
    if (threadIdx.x == 0) scales[r] = s.scale;
    for (int c0 = warp * kShare; c0 < C; c0 += kThreads * 8) {
        k.load(at + c0, C - c0, lane, span, inside);
        k.settle(at + c0, C - c0, lane);
        if (c0 + lane * 8 < C) store_share(k, q + r * q_stride + c0 + lane * 8, s.inverse, C - c0 - lane * 8);
    }
}

template <typename T, Layout kL>
void launch(const exb_ctx* ctx, const T* x, int64_t x_stride, int8_t* q, int64_t q_stride, float* scales, int64_t rows, int C, const Span& span, cudaStream_t st) {
    const int64_t shares = ((int64_t)C + kShare - 1) / kShare;
    auto go = [&](auto kernel, int rows_each, int threads = kThreads) {
        launch_overlapped(ctx, kernel, dim3((unsigned)((rows + rows_each - 1) / rows_each)), dim3(threads), st, x, x_stride, q, q_stride, scales, rows, C, span);
    };
    // Few rows are divided among as many warps as have something to do; of many a warp has four shares under way, of one row or of several short ones.
    const bool many = rows * shares > 64 * (int64_t)ctx->sm_count;
    constexpr int kLongest = sizeof(T) == 2 ? 128 : 64;
    if (shares <= 1) many ? go(quantize_whole_rows_kernel<T, kL, 1, 1, 4>, 32) : go(quantize_whole_rows_kernel<T, kL, 1, 1, 1>, 8);
    else if (shares <= 2) many ? go(quantize_whole_rows_kernel<T, kL, 1, 2, 2>, 16) : go(quantize_whole_rows_kernel<T, kL, 2, 1, 1>, 4);
    else if (shares <= 4) many ? go(quantize_whole_rows_kernel<T, kL, 1, 4, 1>, 8) : go(quantize_whole_rows_kernel<T, kL, 4, 1, 1>, 2);
    else if (shares <= 8) many ? go(quantize_whole_rows_kernel<T, kL, 2, 4, 1>, 4) : go(quantize_whole_rows_kernel<T, kL, 8, 1, 1>, 1);
    else if (shares <= 16) many ? go(quantize_whole_rows_kernel<T, kL, 4, 4, 1>, 2) : go(quantize_whole_rows_kernel<T, kL, 8, 2, 1>, 1);
    else if (shares <= 32) go(quantize_whole_rows_kernel<T, kL, 8, 4, 1>, 1);
    else if (shares <= 64) go(quantize_whole_rows_kernel<T, kL, 8, 8, 1>, 1);
    else if (shares <= kLongest) go(quantize_whole_rows_kernel<T, kL, 16, 8, 1>, 1, 512);
    else go(quantize_long_rows_kernel<T, kL>, 1);
}

}  // namespace
}  // namespace exb

using namespace exb;

extern "C" int exb_quantize_rows_fwd(exb_ctx* ctx, const exb_rows_desc* d, const void* x, int8_t* q, float* scales, void* stream) {
    EXB_REQUIRE(ctx != nullptr && d != nullptr, "exb_quantize_rows_fwd: null context or descriptor");
    const int in_dtype = d->in_dtype, C = d->C;
    const int64_t n_rows = d->rows, x_stride = d->x_stride, q_stride = d->q_stride;
    const size_t es = rows::element_size(in_dtype);
    EXB_REQUIRE(es != 0, "exb_quantize_rows_fwd: x must be EXB_F16, EXB_BF16 or EXB_F32, got %d", in_dtype);
    EXB_REQUIRE(n_rows >= 0 && C >= 1, "exb_quantize_rows_fwd: bad shape (%lld rows of %d)", (long long)n_rows, C);
    if (n_rows > INT32_MAX || C > INT32_MAX - 65536)
        return fail(EXB_ERR_UNSUPPORTED, "exb_quantize_rows_fwd: %lld rows of %d are too many for one call", (long long)n_rows, C);
    if (n_rows == 0) return EXB_OK;
    EXB_REQUIRE(x && q && scales, "exb_quantize_rows_fwd: null buffer");
    EXB_REQUIRE(x_stride >= C && q_stride >= C, "exb_quantize_rows_fwd: row strides smaller than the rows");
    EXB_REQUIRE(rows::aligned_to(x, es) && rows::aligned_to(scales, 4), "exb_quantize_rows_fwd: x or scales not aligned to its element");
    EXB_REQUIRE(aligned16(q) && q_stride % 16 == 0, "exb_quantize_rows_fwd: q and its row stride must be multiples of 16 bytes");
    const rows::Place in[] = {rows::place_of(x, n_rows, C, x_stride, es)};
    const rows::Place out[] = {rows::place_of(q, n_rows, C, q_stride, 1), rows::place_of(scales, 1, n_rows, n_rows, 4)};
    EXB_REQUIRE(!rows::results_overlap(out, in), "exb_quantize_rows_fwd: a result lies over x or over the other result");
    if (int rc = rows::check_device(ctx, "exb_quantize_rows_fwd")) return rc;
    const bool vec = C % 8 == 0 && rows::vector_rows(x, x_stride, es);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    rows::with_type(in_dtype, [&](auto t) {
        using T = decltype(t);
        const T* in = static_cast<const T*>(x);
        const rows::Span span = rows::span_of(x, n_rows, x_stride, C, es);
        if (vec) launch<T, rows::kVectors>(ctx, in, x_stride, q, q_stride, scales, n_rows, C, span, st);
        else launch<T, rows::kShifted>(ctx, in, x_stride, q, q_stride, scales, n_rows, C, span, st);
    });
    return after_launch("exb_quantize_rows_fwd");
}
