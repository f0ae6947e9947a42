// A step of beam search: the best continuations of every sentence over its beams and the vocabulary.
//   score(j, v) = scores[j] + z[j][v] - log sum exp z[j],  z = scale * logits
// One pass over the rows of logits (logit_rows.cuh, without the entropy) leaves each row's sum and its `top` largest logits, in order: no other token of the
// row can be among a sentence's best.  These are scored in 64 bits, so that what is selected hangs on the sums' 32 bits but not on the
// rounding of scores, and the beams' lists are merged by a warp.  Beams that have ended or are none (a score of minus infinity) are not read.
// The CTAs of a sentence are a cluster, whose first one has the lists in its shared memory and merges them; with more beams than a cluster has CTAs,
// and for rows so short that a warp has one, the lists go through a workspace to a second kernel.
// 128 x 8 rows of 131072 fp16 take 58.8 us with 8 selected (4570 GB/s), 64 x 5 of 50001 bf16 18.8, 4 of 131072 fp32 9.4.  Bound by the waits
// for a row's batches of logits and by its end: 39 % of the issue slots are used, 64 % of the exponentials' unit, 70 % of the copy rate.
#include <algorithm>

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

struct Answer {
    float* scores;
    int32_t *parents, *tokens;
    int beams, select, end_token;
};
struct MergeArgs {
    BeamArgs rows;
    Answer to;
};

// Scores in an order of unsigned numbers: NaN above all; 0 is none.
__device__ __forceinline__ unsigned long long order_of(double v) {
    if (v != v) return ~0ull;
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}

// A logit's score; minus infinity: none.  sum: the row's largest logit and log2 of the sum about it.
__device__ __forceinline__ double score_of(float before, float2 sum, float x, float scale) {
    if (sum.y != sum.y) return NAN;
    if (x == -INFINITY) return -INFINITY;
    return (double)before + (((double)x - (double)sum.x) * (double)scale - (double)sum.y * 0.69314718055994530942);
}

// The best of up to 32 falling lists, one a lane, taken `select` times by a warp: 60 ns each.  (Every candidate's place by a search in each list took
// 74 us for 32 beams and 32 selected, and 5 for 4 beams and 8.)  at(list, place): the order of a score (0: none); before(i, j, place_i, place_j): of two lists whose
// heads have equal scores, whether i's comes first.  Lane s ends up with the s-th best: its list, or -1, and its place in that.
template <typename At, typename Before>
__device__ __forceinline__ int2 merge_lists(int lists, int top, int select, int lane, At&& at, Before&& before) {
    int place = 0;
    int2 won = make_int2(-1, 0);
    unsigned long long head = lane < lists ? at(lane, 0) : 0;
    for (int s = 0; s < select; ++s) {
        const uint32_t hi = (uint32_t)(head >> 32), best = __reduce_max_sync(0xffffffffu, hi);
        if (best == 0) break;      // (no score's upper half is 0)
        const uint32_t lo = hi == best ? (uint32_t)head : 0, low = __reduce_max_sync(0xffffffffu, lo);
        uint32_t equal = __ballot_sync(0xffffffffu, hi == best && lo == low);
        int winner = __ffs(equal) - 1;
        for (equal &= equal - 1; equal; equal &= equal - 1) {
            const int other = __ffs(equal) - 1;
            const int mine = __shfl_sync(0xffffffffu, place, winner), theirs = __shfl_sync(0xffffffffu, place, other);
            if (before(other, winner, theirs, mine)) winner = other;
        }
        const int of = __shfl_sync(0xffffffffu, place, winner);
        if (lane == s) won = make_int2(winner, of);
        if (lane == winner) {
            ++place;
            head = place < top ? at(lane, place) : 0;
        }
    }
    return won;
}

__device__ __forceinline__ void answer(const Answer& to, int64_t sentence, int lane, bool is, double score, int parent, int token) {
    if (lane >= to.select) return;
    const int64_t at = sentence * to.select + lane;
    to.scores[at] = is ? (float)score : -INFINITY;
    to.parents[at] = is ? parent : -1;
    to.tokens[at] = is ? token : -1;
}

// ---- a cluster for a sentence --------------------------------------------------------------------
// CTA r of the cluster has part r % splits of beam r / splits.
constexpr int kMostCtas = 16;

struct SentenceArgs {
    const void* logits;
    const float* scores;
    const uint8_t* ended;
    int64_t stride;
    int V, top, splits;
    float scale;
    Answer to;
};

// What slow_row writes to: one beam's sum and list.
struct SlowArgs {
    int V, top;
    float scale;
    float2* sum;
    unsigned long long* best;
    __device__ __forceinline__ void row_is(int64_t, const Row& r) const { *sum = r.empty ? make_float2(0.f, INFINITY) : make_float2(r.m, r.log_s); }
    template <typename T>
    __device__ __forceinline__ void given(const T*, int64_t, const Row&, int, int) const {}
    __device__ __forceinline__ void best_is(int64_t, int place, int token, float logit, const Row&) const { best[place] = key_of(logit, token); }
};

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == kNarrow ? 4 : 2) beam_sentence_kernel(const __grid_constant__ SentenceArgs a) {
    __shared__ Shared<kThreads> sh;
    // (of the cluster's CTAs, in the first one)
    __shared__ Sums s_sums[kMostCtas];
    __shared__ int s_too_many[kMostCtas];
    __shared__ unsigned long long s_best[kMostCtas * kMaxTop], s_order[kMostCtas * kMaxTop];
    __shared__ float2 s_row[kMostCtas];
    __shared__ float s_before[kMostCtas];
    __shared__ int s_state[kMostCtas];      // of a beam
    enum { kNormal, kNone, kEnded, kUnknown, kTooMany };
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int splits = a.splits, beams = a.to.beams, ctas = beams * splits, top = a.top;
    const int64_t sentence = blockIdx.x / ctas;
    const int rank = (int)(blockIdx.x - sentence * ctas), beam = rank / splits, part_of = rank - beam * splits;
    const float c = a.scale * kLog2e;
    auto row_at = [&](int j) { return static_cast<const T*>(a.logits) + (sentence * beams + j) * a.stride; };
    const T* x = row_at(beam);
    const Parts<T> part(x, a.V);
    const int lo = (int)((int64_t)part_of * part.vecs / splits), hi = (int)((int64_t)(part_of + 1) * part.vecs / splits);
    if (tid == 0) {
        sh.n_list = 0;
        sh.n_threads = 0;
        sh.tau = 0;
    }
    __syncwarp();
    ptx::cluster_arrive();      // (waited for before anything is written into the first CTA)
    pdl_enter();
    const float before = a.scores[sentence * beams + beam];
    const bool ended = a.ended && a.ended[sentence * beams + beam];
    if (before != -INFINITY && !ended) {
        const PartSeen seen = see_part<T, kThreads, false>(
            x, part, c, top, lo, hi, part_of == 0 ? part.head : 0, part_of == splits - 1 ? a.V - part.tail0 : 0, sh,
            [&] {
                __syncwarp();
                ptx::cluster_wait();
            },
            [&](int place, unsigned long long key) { ptx::st_cta_u64(ptx::map_to_cta(ptx::smem_u32(&s_best[rank * top + place]), 0), key); });
        if (tid == 0) {
            const uint32_t to = ptx::map_to_cta(ptx::smem_u32(&s_sums[rank]), 0);
            ptx::st_cta_u64(to, (unsigned long long)__float_as_uint(seen.all.s) << 32 | __float_as_uint(seen.all.e));
            ptx::st_cta_u64(to + 8, (unsigned long long)__float_as_uint(seen.all.m) << 32 | __float_as_uint(seen.all.w));
            ptx::st_cta_u32(ptx::map_to_cta(ptx::smem_u32(&s_too_many[rank]), 0), seen.too_many ? 1u : 0u);
        }
    } else {
        __syncwarp();
        ptx::cluster_wait();
    }
    __syncwarp();
    ptx::cluster_sync();
    if (rank) return;
    // the beams' sums, a thread each
    if (tid < beams) {
        const float score = a.scores[sentence * beams + tid];
        int state = kNormal;
        s_before[tid] = score;
        if (score == -INFINITY) {
            state = kNone;
        } else if (a.ended && a.ended[sentence * beams + tid]) {
            state = kEnded;
        } else {
            Sums all = s_sums[tid * splits];
            bool too_many = s_too_many[tid * splits] != 0;
            for (int k = 1; k < splits; ++k) {
                const Sums& u = s_sums[tid * splits + k];
                const float e = fmaxf(all.e, u.e);      // (a part without anything has e = -inf and s = 0)
                if (e != -INFINITY) all.s = all.s * exp2_fast(fmaxf(all.e - e, -1000.f)) + u.s * exp2_fast(fmaxf(u.e - e, -1000.f));
                else all.s += u.s;
                all.e = e;
                all.m = max_nan(all.m, u.m);
                too_many = too_many || s_too_many[tid * splits + k] != 0;
            }
            if (!row_known<T>(all, c)) {
                state = kUnknown;
            } else {
                const Row r = row_of(all, a.scale);
                s_row[tid] = make_float2(r.m, r.log_s);
                if (too_many) state = kTooMany;
            }
        }
        s_state[tid] = state;
    }
    __syncthreads();
    for (int j = 0; j < beams; ++j) {      // (rarely any)
        const int state = s_state[j];
        if (state != kUnknown && state != kTooMany) continue;
        for (int i = tid; i < splits * top; i += kThreads) s_best[j * splits * top + i] = 0;
        __syncthreads();
        const SlowArgs slow = {a.V, top, a.scale, &s_row[j], &s_best[j * splits * top]};
        slow_row<T, kThreads>(slow, row_at(j), 0, sh.part_f, &sh.tau, state == kTooMany, Row{s_row[j].x, s_row[j].y, 0.f, false, a.scale});
        __syncthreads();
    }
    for (int i = tid; i < ctas * top; i += kThreads) {
        const int list = i / top, j = list / splits, state = s_state[j];
        double v = -INFINITY;
        if (state == kEnded) {
            if (i == j * splits * top) v = s_before[j];
        } else if (state != kNone) {
            const unsigned long long key = s_best[i];
            if (key) v = score_of(s_before[j], s_row[j], logit_of(key), a.scale);
        }
        s_order[i] = v == -INFINITY ? 0 : order_of(v);
    }
    __syncthreads();
    if (warp) return;
    // (of equal scores the lower beam's; a beam's by their logits)
    const int2 won = merge_lists(
        ctas, top, a.to.select, lane, [&](int list, int place) { return s_order[list * top + place]; },
        [&](int i, int j, int at_i, int at_j) { return i / splits == j / splits ? s_best[i * top + at_i] > s_best[j * top + at_j] : i < j; });
    const bool is = won.x >= 0;
    const int j = is ? won.x / splits : 0;
    const unsigned long long key = is && s_state[j] != kEnded ? s_best[won.x * top + won.y] : 0;
    answer(a.to, sentence, lane, is, !is ? 0.0 : s_state[j] == kEnded ? (double)s_before[j] : score_of(s_before[j], s_row[j], logit_of(key), a.scale), j,
           is && s_state[j] == kEnded ? a.to.end_token : index_of(key));
}

// ---- through a workspace -------------------------------------------------------------------------
constexpr int kMergeThreads = 128;

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const __grid_constant__ MergeArgs a) {
    __shared__ unsigned long long keys[kMaxBeams * kMaxTop];
    pdl_enter();
    const int tid = threadIdx.x, lane = tid & 31, top = a.rows.top, n = a.to.beams * top;
    const int64_t first = (int64_t)blockIdx.x * a.to.beams;
    auto score_at = [&](int beam, int place) -> double {      // minus infinity: none
        const int64_t row = first + beam;
        const float before = a.rows.scores[row];
        const bool ended = a.rows.ended && a.rows.ended[row];
        const float2 sum = a.rows.sums[row];                                      // (of a row that was left out: whatever was there)
        const float x = __int_as_float(a.rows.best[row * top + place].x);
        if (before == -INFINITY) return -INFINITY;
        if (ended) return place ? -INFINITY : before;
        return score_of(before, sum, x, a.rows.scale);
    };
    for (int i = tid; i < n; i += kMergeThreads) {
        const int beam = i / top;
        const double v = score_at(beam, i - beam * top);
        keys[i] = v == -INFINITY ? 0 : order_of(v);
    }
    __syncthreads();
    if (tid >= 32) return;
    const int2 won = merge_lists(a.to.beams, top, a.to.select, lane, [&](int list, int place) { return keys[list * top + place]; },
                                 [](int i, int j, int, int) { return i < j; });
    double v = 0.0;
    int token = -1;
    if (won.x >= 0) {
        v = score_at(won.x, won.y);
        token = a.rows.ended && a.rows.ended[first + won.x] ? a.to.end_token : a.rows.best[(first + won.x) * top + won.y].y;
    }
    answer(a.to, blockIdx.x, lane, won.x >= 0, v, won.x, token);
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
    EXB_REQUIRE(logits && scores && out_scores && parents && tokens, "exb_beam_select_fwd: null buffer");
    EXB_REQUIRE(!ended || (d->end_token >= 0 && d->end_token < V), "exb_beam_select_fwd: end token %d of %d", d->end_token, V);
    EXB_REQUIRE(stride >= V, "exb_beam_select_fwd: row stride smaller than the rows");
    EXB_REQUIRE(!workspace || d->workspace_bytes >= workspace_of(n_rows, top), "exb_beam_select_fwd: the workspace has %lld bytes, %lld are needed", (long long)d->workspace_bytes,
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
    const Answer to = {out_scores, parents, tokens, beams, select, d->end_token};
    const RowPlan plan = plan_rows(ctx->sm_count, n_rows, (int64_t)V * (int64_t)es);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int rc = EXB_OK;
    // A cluster for a sentence saves a launch and what the second kernel waits for, but its CTAs wait for each other: with rows for more than one wave of CTAs that
    // costs more (us, one kernel and two: 4 x 131072 fp32 9.3 and 9.4, 16 x 4 x 32000 bf16 9.7 and 11.3, 8 x 16 x 131072 fp16 with 32 selected 26.6 and 32.9, 54 x 9 x
    // 11037 fp16 15.2 and 15.7, 64 x 8 x 131072 fp32 58 and 60; 80 x 8 x 131072 fp16 49.5 and 45.9, 100 x 8 x 50000 30.1 and 27.4, 128 x 8 x 131072 61.5 and 60.3, 60 x 16
    // x 32000 bf16 with 32 selected 45 and 37; since a row's second look is in place both take 1 to 3 % less).
    // Few rows with many beams have fewer and longer parts in a cluster: 100 KB more in each cost about what the second kernel does (rows of 524 KB,
    // 131072 fp32, in one kernel and in two: 4 beams 131 and 66 KB 9.2 and 10.1, 5 beams 175 and 66 KB 10.8 and 10.7, 8 beams 262 and 66 KB 13.8 and 12.9, 10 beams 524
    // and 66 KB 19.8 and 16.0), on the device.  60 KB more are allowed for: a call of two kernels takes the host 4 us longer, though not one that has been captured.
    const int64_t bytes = (int64_t)V * (int64_t)es;
    const int parts = std::min(plan.splits, std::max(1, kMostCtas / beams));
    if (!plan.warps && beams <= kMostCtas && 2 * n_rows <= 7 * ctx->sm_count && bytes / parts - bytes / plan.splits <= 160000) {
        SentenceArgs a = {logits, scores, ended, stride, V, top, parts, d->scale, to};
        const unsigned ctas = (unsigned)(beams * a.splits);
        rows::with_type(dtype, [&](auto t) {
            using T = decltype(t);
            auto go = [&](auto threads) {
                constexpr int kThreads = decltype(threads)::value;
                const auto kernel = beam_sentence_kernel<T, kThreads>;
                if (ctas > 8)
                    if (int e = allow_wide_clusters(ctx, kernel)) return e;
                return launch_pdl_cluster(ctx, "beam_sentence_kernel", kernel, dim3((unsigned)sentences * ctas), dim3(kThreads), dim3(ctas), 0, st, a);
            };
            rc = plan.wide ? go(std::integral_constant<int, kWide>()) : go(std::integral_constant<int, kNarrow>());
        });
        return rc;
    }
    if (!workspace) return fail(EXB_ERR_NOMEM, "exb_beam_select_fwd: %d beams of %d tokens need a workspace of %lld bytes", beams, V, (long long)workspace_of(n_rows, top));
    MergeArgs m;
    m.to = to;
    BeamArgs& a = m.rows;
    a.logits = logits; a.scores = scores; a.ended = ended;
    a.sums = static_cast<float2*>(workspace);
    a.best = reinterpret_cast<int2*>(a.sums + n_rows);
    a.stride = stride; a.V = V; a.top = top; a.scale = d->scale; a.splits = plan.splits;
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
