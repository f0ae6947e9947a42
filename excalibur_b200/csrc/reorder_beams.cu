// The states of beams follow their parents, in place: after a step of beam search row j of a sentence's rows becomes what row parents[j] was.
// A thread has the same few bytes of all of a sentence's rows: it reads those of the parents of beams that change, and only then writes, so that
// no row is lost whatever the parents are, and no other thread is waited for.  Beams that are their own parents are neither read nor written
// (but as another's parent), nor are positions from the sentence's length on.
// Bound by memory: the beams that change, in and out once.  us (of them at the copy rate): 4 beams of which 2 change, 64 states of 8 x 512 positions x 128 fp16, 42
// (41); 16 x 8 beams, 6 change, 16 states of 8 x 1024 to 2047 positions x 64 bf16, 665 (737: parents that several beams have are in L2); rows that start anywhere go
// in units of what divides them: 2 x 5 beams, 43 channels in fp32, 75 (54), 4 x 8 beams, 37 channels in fp16, 15 (7).
#include <algorithm>
#include <new>
#include <vector>

#include "rows_common.cuh"

namespace exb {
namespace {

constexpr int kMaxBeams = 32;
constexpr int kMostStates = 1 << 20;
constexpr int kThreads = 256;
constexpr int kStates = 128;           // of one launch
constexpr int kSentences = 256;        // the same

struct ReorderArgs {
    uint8_t* states[kStates];
    const int32_t *parents, *lengths;
    int64_t first;                     // sentence
    int64_t positions, bytes;          // bytes of a position (of all where they follow one another: positions is 1)
    int64_t row_stride, outer_stride, position_stride;
    int64_t outer;
    int64_t per_length;                // positions that follow one another: a sentence's length times this many bytes; otherwise 0
    int n_states, sentences, beams;
};

// A sentence's columns (kUnit bytes of a position, of one state and outer index), in chunks of kThreads * kColumns.
template <typename U, int kColumns>
__device__ __forceinline__ int64_t columns_of(const ReorderArgs& a, int b) {
    const int64_t whole = a.per_length ? a.bytes / a.per_length : a.positions;
    const int64_t length = a.lengths ? min((int64_t)max(a.lengths[a.first + b], 0), whole) : whole;
    return length * ((a.per_length ? a.per_length : a.bytes) / (int64_t)sizeof(U));
}

template <typename U, int kMoves, int kColumns>
__global__ void __launch_bounds__(kThreads) reorder_beams_kernel(const __grid_constant__ ReorderArgs a) {
    __shared__ int s_chunks[kSentences];                        // up to each sentence's end
    __shared__ int64_t s_to[kMaxBeams], s_from[kMaxBeams];      // bytes from the sentence's first row
    __shared__ int s_moves;
    constexpr int kChunk = kThreads * kColumns;
    pdl_enter();
    const int tid = threadIdx.x, lane = tid & 31;
    int mine = 0;
    if (tid < a.sentences) {
        bool moved = false;
        const int32_t* parent = a.parents + (a.first + tid) * a.beams;
        for (int j = 0; j < a.beams; ++j) moved |= parent[j] != j && parent[j] >= 0 && parent[j] < a.beams;
        if (moved) mine = (int)((columns_of<U, kColumns>(a, tid) + kChunk - 1) / kChunk);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, mine, o);
        if (lane >= o) mine += u;
    }
    s_chunks[tid] = mine;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < tid >> 5; ++w) before += s_chunks[w * 32 + 31];
    __syncthreads();
    s_chunks[tid] = mine + before;
    __syncthreads();
    const int chunks = s_chunks[a.sentences - 1];
    const int64_t items = (int64_t)chunks * a.n_states * a.outer;
    int last = -1, moves = 0;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t which = item / chunks;
        const int c = (int)(item - which * chunks);
        int lo = 0, hi = a.sentences - 1;      // the first sentence with more chunks up to its end
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (s_chunks[mid] > c) hi = mid;
            else lo = mid + 1;
        }
        if (lo != last) {
            __syncthreads();
            if (tid < 32) {
                const int p = tid < a.beams ? a.parents[(a.first + lo) * a.beams + tid] : -1;
                const bool moved = p >= 0 && p < a.beams && p != tid;
                const uint32_t all = __ballot_sync(0xffffffffu, moved);
                if (moved) {
                    const int k = __popc(all & ((1u << tid) - 1));
                    s_to[k] = tid * a.row_stride;
                    s_from[k] = p * a.row_stride;
                }
                if (tid == 0) s_moves = __popc(all);
            }
            __syncthreads();
            moves = s_moves;
            last = lo;
        }
        const int64_t outer = which % a.outer;
        uint8_t* base = a.states[which / a.outer] + outer * a.outer_stride + (a.first + lo) * a.beams * a.row_stride;
        const int64_t columns = columns_of<U, kColumns>(a, lo), per = a.bytes / (int64_t)sizeof(U);
        const int64_t column0 = (int64_t)(c - (lo ? s_chunks[lo - 1] : 0)) * kChunk + tid;
        uint8_t* at[kColumns];
#pragma unroll
        for (int k = 0; k < kColumns; ++k) {
            const int64_t column = column0 + k * kThreads;
            at[k] = nullptr;
            if (column < columns) {
                const int64_t position = a.positions > 1 ? column / per : 0;
                at[k] = base + position * a.position_stride + (column - position * per) * (int64_t)sizeof(U);
            }
        }
        U v[kMoves][kColumns];
#pragma unroll
        for (int i = 0; i < kMoves; ++i) {
            if (i >= moves) break;
            const int64_t from = s_from[i];
#pragma unroll
            for (int k = 0; k < kColumns; ++k)
                if (at[k]) v[i][k] = *reinterpret_cast<const U*>(at[k] + from);
        }
#pragma unroll
        for (int i = 0; i < kMoves; ++i) {
            if (i >= moves) break;
            const int64_t to = s_to[i];
#pragma unroll
            for (int k = 0; k < kColumns; ++k)
                if (at[k]) *reinterpret_cast<U*>(at[k] + to) = v[i][k];
        }
    }
}

// ---- host: where states lie ----------------------------------------------------------------------
struct Dim {
    int64_t n, stride;
};
// Sizes and strides that states of a call have, from the outermost in, each dimension inside one step of the next outer one.
struct Layout {
    std::vector<Dim> dims;
    int64_t bytes, extent;      // side by side; from the first byte to behind the last
};
struct State {
    const uint8_t* at;
    int32_t layout;
};
// false where some rows lie over others
bool nest(const exb_reorder_desc& d, Layout& to) {
    to.dims.clear();
    for (const Dim& x : {Dim{d.sentences * d.beams, d.row_stride}, Dim{d.outer, d.outer_stride}, Dim{d.positions, d.position_stride}})
        if (x.n > 1) to.dims.push_back(x);
    std::sort(to.dims.begin(), to.dims.end(), [](const Dim& a, const Dim& b) { return a.stride > b.stride; });
    to.bytes = to.extent = d.bytes;
    for (size_t i = to.dims.size(); i-- > 0;) {
        if (to.dims[i].stride < to.extent) return false;
        to.extent += (to.dims[i].n - 1) * to.dims[i].stride;
    }
    return true;
}

// Whether two states share a byte whose first ones are `d` apart.  Steps of either are taken from the longest stride on (one that both have: as many as one is
// ahead of the other), in every number that leaves them within reach of each other: two at most where their dimensions lie inside each other's steps.
// Where they do not, that can be many: states that `steps` do not suffice for count as sharing memory.
bool meet(const Layout& a, size_t i, const Layout& b, size_t j, int64_t a_extent, int64_t b_extent, int64_t d, int& steps) {
    if (d >= a_extent || -d >= b_extent) return false;
    if (i == a.dims.size() && j == b.dims.size()) return true;      // (the extents are the bytes)
    if (--steps < 0) return true;
    const bool of_a = i < a.dims.size() && (j == b.dims.size() || a.dims[i].stride >= b.dims[j].stride);
    const bool of_b = j < b.dims.size() && (i == a.dims.size() || b.dims[j].stride >= a.dims[i].stride);
    const int64_t stride = of_a ? a.dims[i].stride : b.dims[j].stride, n_a = of_a ? a.dims[i].n : 1, n_b = of_b ? b.dims[j].n : 1;
    a_extent -= (n_a - 1) * stride;
    b_extent -= (n_b - 1) * stride;
    auto floor_of = [&](int64_t v) { return v >= 0 ? v / stride : -((-v + stride - 1) / stride); };
    const int64_t from = std::max(-(n_b - 1), floor_of(d - a_extent) + 1), to = std::min(n_a - 1, floor_of(d + b_extent - 1));      // d - s * stride below a_extent, above -b_extent
    for (int64_t s = from; s <= to; ++s)
        if (meet(a, i + of_a, b, j + of_b, a_extent, b_extent, d - s * stride, steps)) return true;
    return false;
}
constexpr int kMostSteps = 4096;

// Whether all of them (sorted) lie side by side within one step of their outermost dimension, as layers inside rows do: then none needs to be looked at with each
// other one.
bool side_by_side(const std::vector<Layout>& layouts, const std::vector<State>& states) {
    const Layout& first = layouts[states[0].layout];
    if (first.dims.empty()) return false;
    const int64_t step = first.dims[0].stride;
    const uint8_t* end = states[0].at;
    for (const State& s : states) {
        const Layout& of = layouts[s.layout];
        if (of.dims.empty() || of.dims[0].stride != step || s.at < end) return false;
        end = s.at + of.extent - (of.dims[0].n - 1) * step;
    }
    return end - states[0].at <= step;
}

// What can be wrong with n calls.  bits: of all addresses, sizes and strides (0: there is nothing to do).
int look_over(const char* what, const exb_reorder_desc* descs, int32_t n, void* const* const* lists, const int32_t* parents, const int32_t* lengths, uintptr_t& bits) {
    bits = 0;
    std::vector<Layout> layouts;
    std::vector<State> states;
    for (int32_t k = 0; k < n; ++k) {
        const exb_reorder_desc& d = descs[k];
        EXB_REQUIRE(d.sentences >= 0 && d.beams >= 1 && d.n_states >= 0 && d.outer >= 0 && d.positions >= 0 && d.bytes >= 0,
                    "%s: bad shape (%lld x %d beams, %d states of %lld x %lld x %lld bytes)", what, (long long)d.sentences, d.beams, d.n_states, (long long)d.outer,
                    (long long)d.positions, (long long)d.bytes);
        if (d.beams > kMaxBeams || d.n_states > kMostStates)
            return fail(EXB_ERR_UNSUPPORTED, "%s: at most %d beams and %d states, got %d and %d", what, kMaxBeams, kMostStates, d.beams, d.n_states);
        if ((double)d.sentences * d.beams * (double)d.outer * (double)d.positions * (double)d.bytes > 274877906944.0)      // 256 GB
            return fail(EXB_ERR_UNSUPPORTED, "%s: states are too large for one call", what);
        if (d.sentences == 0 || d.n_states == 0 || d.outer == 0 || d.positions == 0 || d.bytes == 0) continue;
        EXB_REQUIRE(lists[k] && parents, "%s: null buffer", what);
        EXB_REQUIRE(rows::aligned_to(parents, 4) && rows::aligned_to(lengths, 4), "%s: parents or lengths not aligned to their element", what);
        Layout of;
        EXB_REQUIRE(nest(d, of), "%s: some of a state's rows lie over others", what);
        bits |= (uintptr_t)d.bytes;
        for (const Dim& x : of.dims) bits |= (uintptr_t)x.stride;
        for (int i = 0; i < d.n_states; ++i) {
            const uint8_t* at = static_cast<const uint8_t*>(lists[k][i]);
            EXB_REQUIRE(at, "%s: null state", what);
            auto among = [&](const void* p, int64_t count) {
                const uint8_t* b = static_cast<const uint8_t*>(p);
                return p && b < at + of.extent && b + count * 4 > at;
            };
            EXB_REQUIRE(!among(parents, d.sentences * d.beams) && !among(lengths, d.sentences), "%s: parents or lengths lie among a state's rows", what);
            bits |= reinterpret_cast<uintptr_t>(at);
            states.push_back({at, (int32_t)layouts.size()});
        }
        layouts.push_back(std::move(of));
    }
    if (states.empty()) return EXB_OK;
    // no two share memory
    std::sort(states.begin(), states.end(), [](const State& a, const State& b) { return a.at < b.at; });
    if (side_by_side(layouts, states)) return EXB_OK;
    for (size_t i = 0; i < states.size(); ++i) {
        const Layout& a = layouts[states[i].layout];
        for (size_t j = i + 1; j < states.size() && states[j].at < states[i].at + a.extent; ++j) {
            const Layout& b = layouts[states[j].layout];
            int steps = kMostSteps;
            EXB_REQUIRE(!meet(a, 0, b, 0, a.extent, b.extent, states[j].at - states[i].at, steps), "%s: two states share memory", what);
        }
    }
    return EXB_OK;
}

template <typename U>
int launch(const exb_ctx* ctx, const ReorderArgs& a, int beams, cudaStream_t st) {
    const int64_t columns = a.positions * a.bytes / (int64_t)sizeof(U) * a.sentences * a.n_states * a.outer;
    // A grid of four CTAs an SM (64 states with 2 of 4 beams changed, 4, 6, 8 and 16: 42.1, 46.6, 43.8, 48.7 us), of which their 90 to 194 registers a thread let two, or one,
    // be there at a time.  Values on their way are registers: with 16 bytes each, four columns of up to 4 beams, two of 8, one of more; smaller units take more columns (43 channels in fp32, 1, 2, 4 and 8 columns: 231, 98, 105, 78 us).
    auto go = [&](auto kernel, int each) {
        const int64_t chunks = std::max<int64_t>(1, (columns + each - 1) / each + (int64_t)a.sentences * a.n_states * a.outer);      // at most
        const int64_t grid = std::min<int64_t>(chunks, (int64_t)ctx->sm_count * 4);
        return launch_pdl(ctx, "reorder_beams_kernel", kernel, dim3((unsigned)grid), dim3(kThreads), 0, st, a);
    };
    constexpr bool kVector = sizeof(U) == 16;
    constexpr int c4 = kVector ? 4 : 8, c8 = kVector ? 2 : 8, c16 = kVector ? 1 : 4, c32 = kVector ? 1 : 2;
    if (beams <= 4) return go(reorder_beams_kernel<U, 4, c4>, kThreads * c4);
    if (beams <= 8) return go(reorder_beams_kernel<U, 8, c8>, kThreads * c8);
    if (beams <= 16) return go(reorder_beams_kernel<U, 16, c16>, kThreads * c16);
    return go(reorder_beams_kernel<U, 32, c32>, kThreads * c32);
}

}  // namespace
}  // namespace exb

using namespace exb;

extern "C" int exb_reorder_beams_check(const exb_reorder_desc* d, int32_t n, void* const* const* states, const int32_t* parents, const int32_t* lengths) try {
    EXB_REQUIRE(n >= 0 && (n == 0 || (d && states)), "exb_reorder_beams_check: null descriptors or states");
    uintptr_t bits;
    return look_over("exb_reorder_beams_check", d, n, states, parents, lengths, bits);
} catch (const std::bad_alloc&) {
    return fail(EXB_ERR_NOMEM, "exb_reorder_beams_check: no memory for the list of states");
}

extern "C" int exb_reorder_beams_fwd(exb_ctx* ctx, const exb_reorder_desc* d, void* const* states, const int32_t* parents, const int32_t* lengths, void* stream) try {
    EXB_REQUIRE(ctx != nullptr && d != nullptr, "exb_reorder_beams_fwd: null context or descriptor");
    uintptr_t bits;
    if (int rc = look_over("exb_reorder_beams_fwd", d, 1, &states, parents, lengths, bits)) return rc;
    if (!bits) return EXB_OK;
    if (int rc = rows::check_device(ctx, "exb_reorder_beams_fwd")) return rc;
    ReorderArgs a;
    a.parents = parents; a.lengths = lengths;
    a.row_stride = d->row_stride; a.outer_stride = d->outer_stride; a.position_stride = d->position_stride;
    a.outer = d->outer; a.beams = d->beams;
    a.positions = d->positions; a.bytes = d->bytes; a.per_length = 0;
    if (d->positions == 1 || d->position_stride == d->bytes) {      // positions that follow one another
        a.per_length = d->bytes;
        a.bytes = d->positions * d->bytes;
        a.positions = 1;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    for (a.first = 0; a.first < d->sentences; a.first += kSentences) {
        a.sentences = (int)std::min<int64_t>(kSentences, d->sentences - a.first);
        for (int s = 0; s < d->n_states; s += kStates) {
            a.n_states = std::min(kStates, d->n_states - s);
            for (int i = 0; i < a.n_states; ++i) a.states[i] = static_cast<uint8_t*>(states[s + i]);
            const int rc = bits % 16 == 0 ? launch<uint4>(ctx, a, d->beams, st) : bits % 8 == 0 ? launch<uint2>(ctx, a, d->beams, st) : bits % 4 == 0 ? launch<uint32_t>(ctx, a, d->beams, st)
                         : bits % 2 == 0 ? launch<uint16_t>(ctx, a, d->beams, st) : launch<uint8_t>(ctx, a, d->beams, st);
            if (rc) return rc;
        }
    }
    return EXB_OK;
} catch (const std::bad_alloc&) {
    return fail(EXB_ERR_NOMEM, "exb_reorder_beams_fwd: no memory for the list of %d states", d->n_states);
}
