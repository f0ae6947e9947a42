// A block's result joins the residual stream and the next block's norm is taken of the sum, in one pass:
//   u = norm(h) * post + post_bias,  r = x + residual_scale * gate * u,  n = norm(r) * weight + bias
// A row stays in its threads' registers in fp32 from the loads of h, x and the gate to the stores of r and n (in the
// activations' type, or as e4m3 with a scale for each 128 channels), so that every tensor crosses memory once; the sums of
// the norms are the only thing its warps exchange.  Bound by memory with many rows, by the chain of loads, reductions and
// stores with few.  4096 x 4096 bf16 takes 23.3 us (5760 GB/s), fp32 42.5 (6320 GB/s), bf16 with both norms, a gate and e4m3 29.2
// (4030 GB/s), one row 1.95, 3152 x 1000 fp16 with a gate's rows 6.9; rows that start anywhere (4096 x 1001, 9.1) are loaded and stored in
// single elements.  With everything no unit is full (62 % of the issue slots, 46 % of the warps): a quarter of the stalls are waits for a row's
// loads, as many for the exchanges between lanes and warps in its reductions.
#include "rows_common.cuh"

#include <type_traits>

namespace exb {
namespace {

using namespace rows;

struct NormArgs {
    const void *h, *x, *gate;
    const float *post_weight, *post_bias, *weight, *bias;
    void *r, *n;
    float* n_scales;
    int64_t rows, gate_rows;
    int64_t h_stride, x_stride, gate_stride, r_stride, n_stride, scale_stride;
    int C, quantized;
    float eps, residual_scale;
};

constexpr int kShare = 256;      // elements of a row that a warp holds at a time, 8 in each lane

// Sum over the row's threads: its warp's lanes, then (through shared memory, in the same order everywhere) its warps.  The two
// halves of s_sum take turns, so that one barrier is enough.
template <bool kOneWarp>
__device__ __forceinline__ float row_sum(float v, float (*s_sum)[32], int& turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (!kOneWarp) {
        const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
        if (lane == 0) s_sum[turn][threadIdx.x >> 5] = v;
        __syncthreads();
        v = lane < warps ? s_sum[turn][lane] : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        turn ^= 1;
    }
    return v;
}

// v = norm(v) * weight + bias over the row.  Elements go in pairs, two to an instruction: the number of instructions is
// what the form with both norms, a gate and e4m3 is bound by.
template <bool kLayer, Layout kL, bool kOneWarp, int kPer>
__device__ __forceinline__ void normalise(float2 (&v)[kPer][4], int lane, int share0, int share_step, const NormArgs& a, const float* weight,
                                          const float* bias, float (*s_sum)[32], int& turn) {
    const float inv_c = 1.f / (float)a.C;
    if constexpr (kLayer) {
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s = __fadd2_rn(s, v[i][j]);
        const float mean = row_sum<kOneWarp>(s.x + s.y, s_sum, turn) * inv_c;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {      // (what lies behind the row's end stays 0)
            const int valid = a.C - (share0 + i * share_step) * kShare;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[i][j].x = (kL == kVectors ? lane * 8 : 2 * j * 32 + lane) < valid ? v[i][j].x - mean : 0.f;
                v[i][j].y = (kL == kVectors ? lane * 8 : (2 * j + 1) * 32 + lane) < valid ? v[i][j].y - mean : 0.f;
            }
        }
    }
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s = __ffma2_rn(v[i][j], v[i][j], s);
    const float k = rsqrtf(row_sum<kOneWarp>(s.x + s.y, s_sum, turn) * inv_c + a.eps);
    const float2 kk = make_float2(k, k);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int c0 = (share0 + i * share_step) * kShare, valid = a.C - c0;
        float2 w[4];
        load8_params<kL>(weight + c0, valid, lane, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = __fmul2_rn(__fmul2_rn(v[i][j], kk), w[j]);
        if (bias) {
            load8_params<kL>(bias + c0, valid, lane, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] = __fadd2_rn(v[i][j], w[j]);
        }
    }
}

// kOneWarp: every warp of the CTA has a row of its own; otherwise the CTA has one.  kPer: shares per warp.
constexpr int max_threads(bool one_warp, int per) { return one_warp || per == 1 ? 256 : 512; }

template <typename T, bool kLayer, Layout kL, bool kOneWarp, int kPer>
__global__ void __launch_bounds__(max_threads(kOneWarp, kPer)) residual_norm_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float s_sum[2][32];
    pdl_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = kOneWarp ? (int64_t)blockIdx.x * (blockDim.x >> 5) + warp : blockIdx.x;
    if (kOneWarp && row >= a.rows) return;
    const int share0 = kOneWarp ? 0 : warp, share_step = kOneWarp ? 1 : (int)(blockDim.x >> 5);
    int turn = 0;
    const T* h = static_cast<const T*>(a.h) + row * a.h_stride;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* g = static_cast<const T*>(a.gate) + (a.gate_rows ? row / a.gate_rows : 0) * a.gate_stride;
    // everything is asked for before anything is waited for, as long as there are registers for it
    constexpr bool kAhead = kPer <= 4;
    constexpr int kKept = kAhead ? kPer : 1;
    float2 v[kPer][4];
    Kept<T, kL> hk[kPer], xk[kKept], gk[kKept];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int c0 = (share0 + i * share_step) * kShare, valid = a.C - c0;
        hk[i].load(h + c0, valid, lane);
        if (kAhead && a.x) xk[kAhead ? i : 0].load(x + c0, valid, lane);
        if (kAhead && a.gate) gk[kAhead ? i : 0].load(g + c0, valid, lane);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) hk[i].get(v[i]);
    if (a.post_weight) normalise<kLayer, kL, kOneWarp, kPer>(v, lane, share0, share_step, a, a.post_weight, a.post_bias, s_sum, turn);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int c0 = (share0 + i * share_step) * kShare, valid = a.C - c0;
        constexpr int kAll = kAhead ? 1 : 0;
        if (!kAhead && a.x) xk[0].load(x + c0, valid, lane);
        if (!kAhead && a.gate) gk[0].load(g + c0, valid, lane);
        float2 o[4];
        const float2 scale = make_float2(a.residual_scale, a.residual_scale);
        if (a.gate) {
            gk[i * kAll].get(o);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] = __fmul2_rn(v[i][j], o[j]);
        }
        if (a.x) {
            xk[i * kAll].get(o);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] = __ffma2_rn(scale, v[i][j], o[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] = __fmul2_rn(v[i][j], scale);
        }
        if (a.r) store8<T, kL>(static_cast<T*>(a.r) + row * a.r_stride + c0, valid, lane, v[i]);
    }
    if (!a.n) return;
    normalise<kLayer, kL, kOneWarp, kPer>(v, lane, share0, share_step, a, a.weight, a.bias, s_sum, turn);
    if (a.quantized) {
        uint8_t* q = static_cast<uint8_t*>(a.n) + row * a.n_stride;
        if constexpr (kL == kVectors) {
            float m[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) m[i] = largest_of(v[i]);
            quantize_shares<kPer>(
                [&](int i, float2(&o)[4]) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[j] = v[i][j];
                },
                m, lane, a.scale_stride,
                [&](int i, int& n) {
                    const int c0 = (share0 + i * share_step) * kShare;
                    n = a.C - c0;
                    return q + c0;
                },
                [&](int i) { return a.n_scales + 2 * (share0 + i * share_step) * a.scale_stride + row; });
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int share = share0 + i * share_step, c0 = share * kShare;
                quantize8_strided(v[i], a.C - c0, lane, q + c0, a.n_scales + 2 * share * a.scale_stride + row, a.scale_stride);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int c0 = (share0 + i * share_step) * kShare;
        store8<T, kL>(static_cast<T*>(a.n) + row * a.n_stride + c0, a.C - c0, lane, v[i]);
    }
}

template <typename T, bool kLayer, Layout kL>
int launch(const exb_ctx* ctx, const NormArgs& a, cudaStream_t st) {
    const int shares = (a.C + kShare - 1) / kShare;
    auto go = [&](auto one, auto per) {
        constexpr bool kOne = decltype(one)::value;
        constexpr int kPer = decltype(per)::value;
        const int warps = kOne ? 8 : (shares + kPer - 1) / kPer;
        const int64_t grid = kOne ? (a.rows + warps - 1) / warps : a.rows;
        launch_overlapped(ctx, residual_norm_kernel<T, kLayer, kL, kOne, kPer>, dim3((unsigned)grid), dim3(32 * warps), st, a);
    };
    using Yes = std::true_type;
    using No = std::false_type;
    // Up to two shares a warp has the row and no warp waits for another (bf16, us, with a warp and with a CTA for a row: 1 x 512 1.40 and 1.61,
    // 1024 x 512 3.4 and 3.6, 32768 x 512 21.5 and 34.4).  Wider rows have as many warps as they have shares while those are few (8192 x 1280
    // with a share for a warp 14.6, with two 15.8), then half as many, which exchange their sums sooner (8192 wide: 64 rows 3.6, in
    // single shares 3.8, in four 3.9; 2048 rows 25.7, 26.2, 27.6; 4096 x 4096 with everything 29.2, 30.9, 31.0; one row of 4096 1.93, 1.86).
    // A CTA has 16 warps, so that a thread may have 128 registers: four shares for a warp beyond 8192, eight beyond 16384.
    if (shares == 1) go(Yes(), std::integral_constant<int, 1>());
    else if (shares == 2) go(Yes(), std::integral_constant<int, 2>());
    else if (shares <= 8) go(No(), std::integral_constant<int, 1>());
    else if (shares <= 32) go(No(), std::integral_constant<int, 2>());
    else if (shares <= 64) go(No(), std::integral_constant<int, 4>());
    else go(No(), std::integral_constant<int, 8>());
    return after_launch("exb_residual_norm_fwd");
}

}  // namespace
}  // namespace exb

using namespace exb;

extern "C" int exb_residual_norm_fwd(exb_ctx* ctx, const exb_norm_desc* d, const void* h, const void* x, const float* post_weight,
                                     const float* post_bias, const void* gate, const float* weight, const float* bias, void* r, void* n,
                                     float* n_scales, void* stream) {
    EXB_REQUIRE(ctx != nullptr && d != nullptr, "exb_residual_norm_fwd: null context or descriptor");
    const size_t es = rows::element_size(d->dtype);
    EXB_REQUIRE(es != 0, "exb_residual_norm_fwd: dtype must be EXB_F16, EXB_BF16 or EXB_F32, got %d", d->dtype);
    const bool quantized = d->out_dtype == EXB_E4M3;
    EXB_REQUIRE(quantized || d->out_dtype == d->dtype, "exb_residual_norm_fwd: the norm is written in dtype or as EXB_E4M3, got %d", d->out_dtype);
    EXB_REQUIRE(d->kind == EXB_NORM_RMS || d->kind == EXB_NORM_LAYER, "exb_residual_norm_fwd: norm %d is not known", d->kind);
    EXB_REQUIRE(d->rows >= 0 && d->C >= 1, "exb_residual_norm_fwd: bad shape (%lld rows of %d)", (long long)d->rows, d->C);
    EXB_REQUIRE(d->eps >= 0.f, "exb_residual_norm_fwd: eps must not be negative");
    if (d->C > 32768 || d->rows > INT32_MAX)
        return fail(EXB_ERR_UNSUPPORTED, "exb_residual_norm_fwd: at most 32768 channels and 2^31 - 1 rows, got %lld rows of %d", (long long)d->rows, d->C);
    if (d->rows == 0) return EXB_OK;
    if (int rc = rows::check_device(ctx, "exb_residual_norm_fwd")) return rc;
    EXB_REQUIRE(h && (r || n), "exb_residual_norm_fwd: null buffer");
    EXB_REQUIRE(!n || weight, "exb_residual_norm_fwd: the norm has no weight");
    EXB_REQUIRE(!post_bias || post_weight, "exb_residual_norm_fwd: a bias without its norm's weight");
    EXB_REQUIRE(d->gate_rows >= 0, "exb_residual_norm_fwd: gate_rows must not be negative");
    EXB_REQUIRE(d->h_stride >= d->C && (!x || d->x_stride >= d->C) && (!r || d->r_stride >= d->C) && (!n || d->n_stride >= d->C),
                "exb_residual_norm_fwd: row strides smaller than the rows");
    EXB_REQUIRE(!gate || d->gate_rows == 0 || d->gate_stride >= d->C, "exb_residual_norm_fwd: row stride of the gate smaller than its rows");
    for (const void* p : {h, x, gate, static_cast<const void*>(r), static_cast<const void*>(quantized ? nullptr : n)})
        EXB_REQUIRE(rows::aligned_to(p, es), "exb_residual_norm_fwd: a tensor is not aligned to its element");
    for (const float* p : {post_weight, post_bias, weight, bias, static_cast<const float*>(n_scales)})
        EXB_REQUIRE(rows::aligned_to(p, 4), "exb_residual_norm_fwd: a parameter is not aligned to its element");
    if (n && quantized) {
        EXB_REQUIRE(n_scales && d->scale_stride >= d->rows, "exb_residual_norm_fwd: null n_scales, or a scale stride smaller than the rows");
        EXB_REQUIRE(aligned16(n) && d->n_stride % 16 == 0, "exb_residual_norm_fwd: e4m3 rows must start at multiples of 16 bytes");
    }
    {
        // r and n may take h's or x's own place, where a row's threads read it before they write it; over any other input, or part of one, a
        // row would be read after another has written it.
        const int64_t gates = d->gate_rows ? (d->rows - 1) / d->gate_rows + 1 : 1;
        const int64_t blocks = (d->C + rows::kBlock - 1) / rows::kBlock;
        const rows::Place in[] = {rows::place_of(h, d->rows, d->C, d->h_stride, es),     rows::place_of(x, d->rows, d->C, d->x_stride, es),
                                  rows::place_of(gate, gates, d->C, d->gate_stride, es), rows::place_of(post_weight, 1, d->C, d->C, 4),
                                  rows::place_of(post_bias, 1, d->C, d->C, 4),           rows::place_of(n ? weight : nullptr, 1, d->C, d->C, 4),
                                  rows::place_of(n ? bias : nullptr, 1, d->C, d->C, 4)};
        const rows::Place out[] = {rows::place_of(r, d->rows, d->C, d->r_stride, es), rows::place_of(n, d->rows, d->C, d->n_stride, quantized ? 1 : es),
                                   rows::place_of(n && quantized ? n_scales : nullptr, blocks, d->rows, d->scale_stride, 4)};
        for (int i = 0; i < 3; ++i) {
            for (int j = 0; j < 7; ++j)
                EXB_REQUIRE(!rows::overlap(out[i], in[j]) || (i < 2 && j < 2 && rows::same_place(out[i], in[j])),
                            "exb_residual_norm_fwd: a result lies over an input (r and n may take the place of h or x, with its stride)");
            for (int j = 0; j < i; ++j) EXB_REQUIRE(!rows::overlap(out[i], out[j]), "exb_residual_norm_fwd: results lie over each other");
        }
    }
    NormArgs a;
    a.h = h; a.x = x; a.gate = gate;
    a.post_weight = post_weight; a.post_bias = post_bias; a.weight = weight; a.bias = bias;
    a.r = r; a.n = n; a.n_scales = n_scales;
    a.rows = d->rows; a.gate_rows = d->gate_rows;
    a.h_stride = d->h_stride; a.x_stride = d->x_stride; a.gate_stride = d->gate_rows ? d->gate_stride : 0;
    a.r_stride = d->r_stride; a.n_stride = d->n_stride; a.scale_stride = d->scale_stride;
    a.C = d->C; a.quantized = quantized;
    a.eps = d->eps; a.residual_scale = d->residual_scale;
    bool vec = d->C % 8 == 0 && rows::vector_rows(h, d->h_stride, es) && rows::vector_rows(x, d->x_stride, es) &&
               rows::vector_rows(gate, a.gate_stride, es) && rows::vector_rows(r, d->r_stride, es) && (quantized || rows::vector_rows(n, d->n_stride, es));
    for (const float* p : {post_weight, post_bias, weight, bias}) vec = vec && aligned16(p);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int rc = EXB_OK;
    rows::with_type(d->dtype, [&](auto t) {
        using T = decltype(t);
        if (d->kind == EXB_NORM_LAYER) rc = vec ? launch<T, true, rows::kVectors>(ctx, a, st) : launch<T, true, rows::kStrided>(ctx, a, st);
        else rc = vec ? launch<T, false, rows::kVectors>(ctx, a, st) : launch<T, false, rows::kStrided>(ctx, a, st);
    });
    return rc;
}
