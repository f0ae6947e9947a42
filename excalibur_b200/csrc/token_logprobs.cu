// Log probabilities of given tokens, the entropy and the most probable tokens of rows of logits.
//
// z = scale * x, p = exp(z - lse), lse = log sum exp z.  With any e, t = x * scale * log2(e) - e, s = sum 2^t, w = sum 2^t * t:
//   log p(v) = ln 2 * (t_v - log2 s),  entropy = ln 2 * (log2 s - w / s).
// One pass over the row, bound by its reading and, in 16 bits, by the latency of its loads (50 % of the issue slots are used, 40 to
// 46 % of the warps' stalls are waits for logits, and a CTA's loads drain at its row's end): 2048 rows of 50001 fp16 take 42.4 us with the
// top 5 (4830 GB/s), 37.0 without, 49.6 with 20; 1024 rows of 50000 fp32 without 33.5 (6110 GB/s); one row of 131072 fp32 with 20 7.1.
#include "logit_rows.cuh"

namespace exb {
namespace {

using namespace logits;

struct LogprobArgs {
    const void* logits;
    const int32_t* tokens;
    float *logprobs, *entropy, *top_logprobs;
    int32_t* top_tokens;
    int64_t stride;
    int V, n_given, top, splits;
    float scale;

    static constexpr bool kEntropy = true;
    __device__ __forceinline__ bool left_out(int64_t) const { return false; }
    __device__ __forceinline__ void row_is(int64_t row, const Row& r) const {
        if (entropy) entropy[row] = r.entropy;
    }
    template <typename T>
    __device__ __forceinline__ void given(const T* x, int64_t row, const Row& r, int first, int step) const {
        for (int j = first; j < n_given; j += step) {
            const int token = tokens[row * n_given + j];
            logprobs[row * n_given + j] = token < 0 ? 0.f : token >= V ? NAN : r.logprob(to_float<T>(x[token]));
        }
    }
    __device__ __forceinline__ void best_is(int64_t row, int place, int token, float logit, const Row& r) const {
        top_tokens[row * top + place] = token;
        top_logprobs[row * top + place] = r.logprob(logit);
    }
};

template <typename T>
__global__ void __launch_bounds__(kWarpRows * 32) token_logprobs_warp_kernel(const __grid_constant__ LogprobArgs a, int64_t n_rows) {
    rows_by_warps<T>(a, n_rows);
}
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const __grid_constant__ LogprobArgs a) {
    rows_by_ctas<T, kThreads>(a);
}

template <typename T, int kThreads>
int launch(const exb_ctx* ctx, LogprobArgs& a, int64_t n_rows, cudaStream_t st) {
    return launch_pdl_cluster(ctx, "token_logprobs_kernel", token_logprobs_kernel<T, kThreads>, dim3((unsigned)(n_rows * a.splits)), dim3(kThreads), dim3(a.splits), 0,
                              st, a);
}

}  // namespace
}  // namespace exb

using namespace exb;

extern "C" int exb_token_logprobs_fwd(exb_ctx* ctx, const exb_logprobs_desc* d, const void* logits, const int32_t* tokens, float* logprobs,
                                      float* entropy, float* top_logprobs, int32_t* top_tokens, void* stream) {
    EXB_REQUIRE(ctx != nullptr && d != nullptr, "exb_token_logprobs_fwd: null context or descriptor");
    const int64_t n_rows = d->rows, stride = d->stride;
    const int dtype = d->dtype, V = d->V, n_given = d->n_given, top = d->top;
    const float scale = d->scale;
    const size_t es = rows::element_size(dtype);
    EXB_REQUIRE(es != 0, "exb_token_logprobs_fwd: logits must be EXB_F16, EXB_BF16 or EXB_F32, got %d", dtype);
    EXB_REQUIRE(n_rows >= 0 && V >= 1, "exb_token_logprobs_fwd: bad shape (%lld rows of %d)", (long long)n_rows, V);
    EXB_REQUIRE(scale > 1e-8f && scale < 1e8f, "exb_token_logprobs_fwd: scale must be a positive number between 1e-8 and 1e8");
    EXB_REQUIRE(n_given >= 0 && top >= 0, "exb_token_logprobs_fwd: n_given and top must not be negative");
    EXB_REQUIRE(top <= V, "exb_token_logprobs_fwd: %d of %d tokens asked for", top, V);
    if (top > kMaxTop) return fail(EXB_ERR_UNSUPPORTED, "exb_token_logprobs_fwd: at most %d of the most probable tokens, got %d", kMaxTop, top);
    if (n_rows > INT32_MAX / 16 || V > (1 << 30))
        return fail(EXB_ERR_UNSUPPORTED, "exb_token_logprobs_fwd: %lld rows of %d are too many for one call", (long long)n_rows, V);
    if (n_rows == 0) return EXB_OK;
    if (int rc = rows::check_device(ctx, "exb_token_logprobs_fwd")) return rc;
    EXB_REQUIRE(logits && (n_given == 0 || (tokens && logprobs)) && (top == 0 || (top_logprobs && top_tokens)), "exb_token_logprobs_fwd: null buffer");
    EXB_REQUIRE(stride >= V, "exb_token_logprobs_fwd: row stride smaller than the rows");
    EXB_REQUIRE(rows::aligned_to(logits, es), "exb_token_logprobs_fwd: logits not aligned to their element");
    for (const void* p : {static_cast<const void*>(tokens), static_cast<const void*>(logprobs), static_cast<const void*>(entropy),
                          static_cast<const void*>(top_logprobs), static_cast<const void*>(top_tokens)})
        EXB_REQUIRE(rows::aligned_to(p, 4), "exb_token_logprobs_fwd: a buffer is not aligned to its element");
    const rows::Place in[] = {rows::place_of(logits, n_rows, V, stride, es), rows::place_of(n_given ? tokens : nullptr, n_rows, n_given, n_given, 4)};
    const rows::Place out[] = {rows::place_of(n_given ? logprobs : nullptr, n_rows, n_given, n_given, 4), rows::place_of(entropy, 1, n_rows, n_rows, 4),
                               rows::place_of(top ? top_logprobs : nullptr, n_rows, top, top, 4), rows::place_of(top ? top_tokens : nullptr, n_rows, top, top, 4)};
    EXB_REQUIRE(!rows::results_overlap(out, in), "exb_token_logprobs_fwd: a result lies over an input or another result");
    LogprobArgs a;
    a.logits = logits; a.tokens = tokens; a.logprobs = logprobs; a.entropy = entropy; a.top_logprobs = top_logprobs; a.top_tokens = top_tokens;
    a.stride = stride; a.V = V; a.n_given = n_given; a.top = top; a.scale = scale;
    if (n_given == 0 && top == 0 && !entropy) return EXB_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int rc = EXB_OK;
    const RowPlan plan = plan_rows(ctx->sm_count, n_rows, (int64_t)V * (int64_t)es);
    if (plan.warps) {
        rows::with_type(dtype, [&](auto t) {
            using T = decltype(t);
            launch_overlapped(ctx, token_logprobs_warp_kernel<T>, dim3((unsigned)((n_rows + kWarpRows - 1) / kWarpRows)), dim3(kWarpRows * 32), st, a, n_rows);
        });
        return after_launch("token_logprobs_warp_kernel");
    }
    a.splits = plan.splits;
    rows::with_type(dtype, [&](auto t) {
        using T = decltype(t);
        rc = plan.wide ? launch<T, kWide>(ctx, a, n_rows, st) : launch<T, kNarrow>(ctx, a, n_rows, st);
    });
    return rc;
}
