// Log probabilities of given tokens, the entropy and the most probable tokens of rows of logits.
//
// z = scale * x, p = exp(z - lse), lse = log sum exp z.  With M the row's largest logit, t = (x - M) * scale * log2(e),
// s = sum 2^t and w = sum 2^t * t:  log p(v) = ln 2 * (t_v - log2 s),  entropy = ln 2 * (log2 s - w / s).
#include "rows_common.cuh"

namespace exb {
namespace {

using namespace rows;

constexpr int kThreads = 512;
constexpr int kMaxTop = 32;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct LogprobArgs {
    const void* logits;
    const int32_t* tokens;
    float *logprobs, *entropy, *top_logprobs;
    int32_t* top_tokens;
    int64_t stride;
    int V, n_given, top;
    float scale;
};

// Logits in an order of unsigned numbers: both zeros alike, NaN above infinity.  With the index behind it (the lower one is the larger
// key) no two keys are alike.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long key_of(float x, int index) { return (unsigned long long)order_of(x) << 32 | (uint32_t)~index; }

template <typename F>
__device__ __forceinline__ float block_reduce(float v, float* s_part, F op) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s_part[0];
    for (int i = 1; i < kThreads / 32; ++i) v = op(v, s_part[i]);
    return v;
}

// One CTA per row: the maximum, the sums, and a pass over the row for each of the most probable tokens.
template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const __grid_constant__ LogprobArgs a) {
    __shared__ float s_part[kThreads / 32];
    __shared__ unsigned long long s_best;
    pdl_enter();
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    const float c = a.scale * kLog2e;
    float m = -INFINITY;
    for (int i = threadIdx.x; i < a.V; i += kThreads) m = fmaxf(m, to_float<T>(x[i]));
    m = block_reduce(m, s_part, [](float u, float v) { return fmaxf(u, v); });
    float s = 0.f, w = 0.f;
    for (int i = threadIdx.x; i < a.V; i += kThreads) {
        const float v = to_float<T>(x[i]), t = (v - m) * c, p = v == -INFINITY ? 0.f : exp2f(t);
        s += p;
        w += p == 0.f ? 0.f : p * t;
    }
    s = block_reduce(s, s_part, [](float u, float v) { return u + v; });
    w = block_reduce(w, s_part, [](float u, float v) { return u + v; });
    const bool empty = !(s != 0.f);       // (a NaN anywhere makes s one)
    const float log_s = log2f(s);
    // (halves: the distance of fp32's two ends is no fp32 number)
    auto logprob = [&](float v) { return empty ? -INFINITY : (0.5f * v - 0.5f * m) * (2.f * a.scale) - log_s * kLn2; };
    if (threadIdx.x == 0 && a.entropy) a.entropy[row] = empty ? 0.f : (log_s - w / s) * kLn2;
    for (int j = threadIdx.x; j < a.n_given; j += kThreads) {
        const int token = a.tokens[row * a.n_given + j];
        a.logprobs[row * a.n_given + j] = token < 0 ? 0.f : token >= a.V ? NAN : logprob(to_float<T>(x[token]));
    }
    unsigned long long last = ~0ull;
    for (int j = 0; j < a.top; ++j) {
        unsigned long long best = 0;
        for (int i = threadIdx.x; i < a.V; i += kThreads) {
            const unsigned long long k = key_of(to_float<T>(x[i]), i);
            if (k < last && k > best) best = k;
        }
        if (threadIdx.x == 0) s_best = 0;
        __syncthreads();
        atomicMax(&s_best, best);
        __syncthreads();
        last = s_best;
        __syncthreads();
        if (threadIdx.x == 0) {
            const int token = (int)~(uint32_t)last;
            a.top_tokens[row * a.top + j] = token;
            a.top_logprobs[row * a.top + j] = logprob(to_float<T>(x[token]));
        }
    }
}

}  // namespace
}  // namespace exb

using namespace exb;

extern "C" int exb_token_logprobs_fwd(exb_ctx* ctx, const void* logits, int dtype, int64_t stride, int64_t n_rows, int V, float scale,
                                      const int32_t* tokens, int n_given, float* logprobs, float* entropy, int top, float* top_logprobs,
                                      int32_t* top_tokens, void* stream) {
    EXB_REQUIRE(ctx != nullptr, "exb_token_logprobs_fwd: null context");
    const size_t es = rows::element_size(dtype);
    EXB_REQUIRE(es != 0, "exb_token_logprobs_fwd: logits must be EXB_F16, EXB_BF16 or EXB_F32, got %d", dtype);
    EXB_REQUIRE(n_rows >= 0 && V >= 1, "exb_token_logprobs_fwd: bad shape (%lld rows of %d)", (long long)n_rows, V);
    EXB_REQUIRE(scale > 1e-38f && scale < 1e38f, "exb_token_logprobs_fwd: scale must be a positive number");
    EXB_REQUIRE(n_given >= 0 && top >= 0, "exb_token_logprobs_fwd: n_given and top must not be negative");
    EXB_REQUIRE(top <= V, "exb_token_logprobs_fwd: %d of %d tokens asked for", top, V);
    if (top > kMaxTop) return fail(EXB_ERR_UNSUPPORTED, "exb_token_logprobs_fwd: at most %d of the most probable tokens, got %d", kMaxTop, top);
    if (n_rows > INT32_MAX / 16 || V > (1 << 30))
        return fail(EXB_ERR_UNSUPPORTED, "exb_token_logprobs_fwd: %lld rows of %d are too many for one call", (long long)n_rows, V);
    if (n_rows == 0) return EXB_OK;
    EXB_REQUIRE(logits && (n_given == 0 || (tokens && logprobs)) && (top == 0 || (top_logprobs && top_tokens)), "exb_token_logprobs_fwd: null buffer");
    EXB_REQUIRE(stride >= V, "exb_token_logprobs_fwd: row stride smaller than the rows");
    EXB_REQUIRE(rows::aligned_to(logits, es), "exb_token_logprobs_fwd: logits not aligned to their element");
    for (const void* p : {static_cast<const void*>(tokens), static_cast<const void*>(logprobs), static_cast<const void*>(entropy),
                          static_cast<const void*>(top_logprobs), static_cast<const void*>(top_tokens)})
        EXB_REQUIRE(rows::aligned_to(p, 4), "exb_token_logprobs_fwd: a buffer is not aligned to its element");
    LogprobArgs a;
    a.logits = logits; a.tokens = tokens; a.logprobs = logprobs; a.entropy = entropy; a.top_logprobs = top_logprobs; a.top_tokens = top_tokens;
    a.stride = stride; a.V = V; a.n_given = n_given; a.top = top; a.scale = scale;
    if (n_given == 0 && top == 0 && !entropy) return EXB_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    rows::with_type(dtype, [&](auto t) {
        using T = decltype(t);
        launch_overlapped(ctx, token_logprobs_kernel<T>, dim3((unsigned)n_rows), dim3(kThreads), st, a);
    });
    return after_launch("exb_token_logprobs_fwd");
}
