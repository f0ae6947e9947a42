// A step of beam search: the best continuations of every sentence over its beams and the vocabulary.
//   score(j, v) = scores[j] + z[j][v] - log sum exp z[j],  z = scale * logits
// One pass over the rows of logits (logit_rows.cuh, without the entropy) leaves each row's sum and its `top` largest logits, in order: no other token of the
// row can be among a sentence's best.  A second kernel scores those in 64 bits, so that what is selected hangs on the sums' 32 bits
// but not on the rounding of scores, and merges the beams' lists.  Beams that have ended or are none (a score of minus infinity) are not read.
#include "logit_rows.cuh"

namespace exb {
namespace {

using namespace logits;

constexpr int kMaxBeams = 32;

struct BeamArgs {
    const void* logits;
    const float* scores;
    const uint8_t* ended;
    float2* sums;                 // [row] largest logit, log2 of the sum about it
    int2* best;                   // [row][top] logit, token
    int64_t stride;
    int V, top, splits;
    float scale;

    static constexpr bool kEntropy = false;
    __device__ __forceinline__ bool left_out(int64_t row) const { return scores[row] == -INFINITY || (ended && ended[row]); }
    __device__ __forceinline__ void row_is(int64_t row, const Row& r) const { sums[row] = r.empty ? make_float2(0.f, INFINITY) : make_float2(r.m, r.log_s); }
    template <typename T>
    __device__ __forceinline__ void given(const T*, int64_t, const Row&, int, int) const {}
    __device__ __forceinline__ void best_is(int64_t row, int place, int token, float logit, const Row&) const {
        best[row * top + place] = make_int2(__float_as_int(logit), token);
    }
};

template <typename T>
__global__ void __launch_bounds__(kWarpRows * 32) beam_rows_warp_kernel(const __grid_constant__ BeamArgs a, int64_t n_rows) {
    rows_by_warps<T>(a, n_rows);
}
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) beam_rows_kernel(const __grid_constant__ BeamArgs a) {
    rows_by_ctas<T, kThreads>(a);
}

struct MergeArgs {
    BeamArgs rows;
    float* out_scores;
    int32_t *parents, *tokens;
    int beams, select, end_token;
};

// Scores in an order of unsigned numbers: NaN above all; 0 is none.
__device__ __forceinline__ unsigned long long order_of(double v) {
    if (v != v) return ~0ull;
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}

constexpr int kMergeThreads = 128;

// A CTA scores a sentence's candidates; then a lane of its first warp has each beam's list, and the best of the lists' heads is taken `select` times: 60 ns
// each, whatever the number of beams.  (Every candidate's place by a search in each list took 74 us for 32 beams and 32 selected,
// and 5 for 4 beams and 8.)
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const __grid_constant__ MergeArgs a) {
    __shared__ unsigned long long keys[kMaxBeams * kMaxTop];
    pdl_enter();
    const int tid = threadIdx.x, lane = tid & 31, top = a.rows.top, n = a.beams * top;
    const int64_t first = (int64_t)blockIdx.x * a.beams;
    auto score_of = [&](int beam, int place) -> double {      // minus infinity: none
        const int64_t row = first + beam;
        const float before = a.rows.scores[row];
        const bool ended = a.rows.ended && a.rows.ended[row];
        const float2 sum = a.rows.sums[row];                                      // (of a row that was left out: whatever was there)
        const float x = __int_as_float(a.rows.best[row * top + place].x);
        if (before == -INFINITY) return -INFINITY;
        if (ended) return place ? -INFINITY : before;
        if (sum.y != sum.y) return NAN;
        if (x == -INFINITY) return -INFINITY;
        return (double)before + (((double)x - (double)sum.x) * (double)a.rows.scale - (double)sum.y * 0.69314718055994530942);
    };
    for (int i = tid; i < n; i += kMergeThreads) {
        const int beam = i / top;
        const double v = score_of(beam, i - beam * top);
        keys[i] = v == -INFINITY ? 0 : order_of(v);
    }
    __syncthreads();
    if (tid >= 32) return;
    int place = 0, won_beam = -1, won_place = 0;      // this lane's head, and what the lane writes
    const unsigned long long* list = keys + lane * top;
    unsigned long long head = lane < a.beams ? list[0] : 0;
    for (int s = 0; s < a.select; ++s) {
        const uint32_t hi = (uint32_t)(head >> 32), best = __reduce_max_sync(0xffffffffu, hi);
        if (best == 0) break;      // (no score's upper half is 0)
        const uint32_t lo = hi == best ? (uint32_t)head : 0, low = __reduce_max_sync(0xffffffffu, lo);
        const int winner = __ffs(__ballot_sync(0xffffffffu, hi == best && lo == low)) - 1;      // of equal scores the lower beam's
        const int at = __shfl_sync(0xffffffffu, place, winner);
        if (lane == s) {
            won_beam = winner;
            won_place = at;
        }
        if (lane == winner) {
            ++place;
            head = place < top ? list[place] : 0;
        }
    }
    if (lane < a.select) {
        const int64_t at = (int64_t)blockIdx.x * a.select + lane;
        float v = -INFINITY;
        int token = -1;
        if (won_beam >= 0) {
            v = (float)score_of(won_beam, won_place);
            token = a.rows.ended && a.rows.ended[first + won_beam] ? a.end_token : a.rows.best[(first + won_beam) * top + won_place].y;
        }
        a.out_scores[at] = v;
        a.parents[at] = won_beam;
        a.tokens[at] = token;
    }
}

int64_t workspace_of(int64_t n_rows, int top) { return n_rows * (int64_t)(sizeof(float2) + (size_t)top * sizeof(int2)); }

}  // namespace
}  // namespace exb

using namespace exb;

extern "C" int exb_beam_select_fwd(exb_ctx* ctx, const exb_beam_desc* d, const void* logits, const float* scores, const uint8_t* ended, float* out_scores,
                                   int32_t* parents, int32_t* tokens, void* workspace, void* stream) {
    EXB_REQUIRE(ctx != nullptr && d != nullptr, "exb_beam_select_fwd: null context or descriptor");
    const int64_t sentences = d->sentences, stride = d->stride;
    const int beams = d->beams, V = d->V, dtype = d->dtype, select = d->select;
    const size_t es = rows::element_size(dtype);
    EXB_REQUIRE(es != 0, "exb_beam_select_fwd: logits must be EXB_F16, EXB_BF16 or EXB_F32, got %d", dtype);
    EXB_REQUIRE(sentences >= 0 && beams >= 1 && V >= 1 && select >= 1, "exb_beam_select_fwd: bad shape (%lld x %d beams of %d tokens, %d selected)",
                (long long)sentences, beams, V, select);
    EXB_REQUIRE(d->scale > 1e-8f && d->scale < 1e8f, "exb_beam_select_fwd: scale must be a positive number between 1e-8 and 1e8");
    if (beams > kMaxBeams || select > kMaxTop)
        return fail(EXB_ERR_UNSUPPORTED, "exb_beam_select_fwd: at most %d beams and %d selected, got %d and %d", kMaxBeams, kMaxTop, beams, select);
    if (sentences > INT32_MAX / (16 * beams) || V > (1 << 30))
        return fail(EXB_ERR_UNSUPPORTED, "exb_beam_select_fwd: %lld x %d rows of %d are too many for one call", (long long)sentences, beams, V);
    if (sentences == 0) return EXB_OK;
    const int64_t n_rows = sentences * beams;
    const int top = select < V ? select : V;
    EXB_REQUIRE(logits && scores && out_scores && parents && tokens && workspace, "exb_beam_select_fwd: null buffer");
    EXB_REQUIRE(!ended || (d->end_token >= 0 && d->end_token < V), "exb_beam_select_fwd: end token %d of %d", d->end_token, V);
    EXB_REQUIRE(stride >= V, "exb_beam_select_fwd: row stride smaller than the rows");
    EXB_REQUIRE(d->workspace_bytes >= workspace_of(n_rows, top), "exb_beam_select_fwd: the workspace has %lld bytes, %lld are needed", (long long)d->workspace_bytes,
                (long long)workspace_of(n_rows, top));
    EXB_REQUIRE(rows::aligned_to(logits, es) && rows::aligned_to(workspace, 8), "exb_beam_select_fwd: logits or workspace not aligned to their element");
    for (const void* p : {static_cast<const void*>(scores), static_cast<const void*>(out_scores), static_cast<const void*>(parents), static_cast<const void*>(tokens)})
        EXB_REQUIRE(rows::aligned_to(p, 4), "exb_beam_select_fwd: a buffer is not aligned to its element");
    const rows::Place in[] = {rows::place_of(logits, n_rows, V, stride, es), rows::place_of(scores, 1, n_rows, n_rows, 4), rows::place_of(ended, 1, n_rows, n_rows, 1)};
    const int64_t n_out = sentences * select;
    const rows::Place out[] = {rows::place_of(out_scores, 1, n_out, n_out, 4), rows::place_of(parents, 1, n_out, n_out, 4), rows::place_of(tokens, 1, n_out, n_out, 4),
                               rows::place_of(workspace, 1, d->workspace_bytes, d->workspace_bytes, 1)};
    EXB_REQUIRE(!rows::results_overlap(out, in), "exb_beam_select_fwd: a result or the workspace lies over an input or another result");
    if (int rc = rows::check_device(ctx, "exb_beam_select_fwd")) return rc;
    MergeArgs m;
    BeamArgs& a = m.rows;
    a.logits = logits; a.scores = scores; a.ended = ended;
    a.sums = static_cast<float2*>(workspace);
    a.best = reinterpret_cast<int2*>(a.sums + n_rows);
    a.stride = stride; a.V = V; a.top = top; a.scale = d->scale;
    m.out_scores = out_scores; m.parents = parents; m.tokens = tokens; m.beams = beams; m.select = select; m.end_token = d->end_token;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const RowPlan plan = plan_rows(ctx->sm_count, n_rows, (int64_t)V * (int64_t)es);
    a.splits = plan.splits;
    int rc = EXB_OK;
    rows::with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (plan.warps) {
            launch_overlapped(ctx, beam_rows_warp_kernel<T>, dim3((unsigned)((n_rows + kWarpRows - 1) / kWarpRows)), dim3(kWarpRows * 32), st, a, n_rows);
            rc = after_launch("beam_rows_warp_kernel");
        } else {
            const dim3 grid((unsigned)(n_rows * a.splits)), cluster(a.splits);
            rc = plan.wide ? launch_pdl_cluster(ctx, "beam_rows_kernel", beam_rows_kernel<T, kWide>, grid, dim3(kWide), cluster, 0, st, a)
                           : launch_pdl_cluster(ctx, "beam_rows_kernel", beam_rows_kernel<T, kNarrow>, grid, dim3(kNarrow), cluster, 0, st, a);
        }
    });
    if (rc) return rc;
    return launch_pdl(ctx, "beam_merge_kernel", beam_merge_kernel, dim3((unsigned)sentences), dim3(kMergeThreads), 0, st, m);
}
