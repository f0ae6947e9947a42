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
// A state's dimensions from the outermost in, each inside one step of the next outer one; false where some lie over others.
bool nest(const exb_reorder_desc& d, std::vector<Dim>& dims, int64_t& extent) {
    dims.clear();
    for (const Dim& x : {Dim{d.sentences * d.beams, d.row_stride}, Dim{d.outer, d.outer_stride}, Dim{d.positions, d.position_stride}})
        if (x.n > 1) dims.push_back(x);
    std::sort(dims.begin(), dims.end(), [](const Dim& a, const Dim& b) { return a.stride > b.stride; });
    extent = d.bytes;
    for (size_t i = dims.size(); i-- > 0;) {
        if (dims[i].stride < extent) return false;
        extent += (dims[i].n - 1) * dims[i].stride;
    }
    return true;
}
// Whether two states whose first bytes are `d` apart share a byte: at each dimension the step at or before the distance and the one behind it can.
bool meet(const std::vector<Dim>& dims, size_t i, int64_t bytes, int64_t d) {
    if (i == dims.size()) return d < bytes && -d < bytes;
    const int64_t at = d >= 0 ? d / dims[i].stride : -((-d + dims[i].stride - 1) / dims[i].stride);
    for (int64_t s = at; s <= at + 1; ++s)
        if (s < dims[i].n && -s < dims[i].n && meet(dims, i + 1, bytes, d - s * dims[i].stride)) return true;
    return false;
}

// Whether all of them (sorted) lie side by side within one step of the outermost dimension, as layers inside rows do: then none needs to be looked at with each
// other one.
bool side_by_side(const std::vector<Dim>& dims, int64_t extent, const std::vector<const uint8_t*>& at) {
    if (dims.empty()) return false;
    const int64_t inner = extent - (dims[0].n - 1) * dims[0].stride;
    for (size_t i = 1; i < at.size(); ++i)
        if (at[i] - at[i - 1] < inner) return false;
    return at.back() - at.front() + inner <= dims[0].stride;
}

// What can be wrong with a call.  bits: of all addresses, sizes and strides (0: there is nothing to do).
int look_over(const char* what, const exb_reorder_desc& d, void* const* states, const int32_t* parents, const int32_t* lengths, uintptr_t& bits) {
    bits = 0;
    EXB_REQUIRE(d.sentences >= 0 && d.beams >= 1 && d.n_states >= 0 && d.outer >= 0 && d.positions >= 0 && d.bytes >= 0,
                "%s: bad shape (%lld x %d beams, %d states of %lld x %lld x %lld bytes)", what, (long long)d.sentences, d.beams, d.n_states, (long long)d.outer,
                (long long)d.positions, (long long)d.bytes);
    if (d.beams > kMaxBeams || d.n_states > kMostStates)
        return fail(EXB_ERR_UNSUPPORTED, "%s: at most %d beams and %d states, got %d and %d", what, kMaxBeams, kMostStates, d.beams, d.n_states);
    if ((double)d.sentences * d.beams * (double)d.outer * (double)d.positions * (double)d.bytes > 274877906944.0)      // 256 GB
        return fail(EXB_ERR_UNSUPPORTED, "%s: states are too large for one call", what);
    if (d.sentences == 0 || d.n_states == 0 || d.outer == 0 || d.positions == 0 || d.bytes == 0) return EXB_OK;
    EXB_REQUIRE(states && parents, "%s: null buffer", what);
    EXB_REQUIRE(rows::aligned_to(parents, 4) && rows::aligned_to(lengths, 4), "%s: parents or lengths not aligned to their element", what);
    std::vector<Dim> dims;
    int64_t extent;
    EXB_REQUIRE(nest(d, dims, extent), "%s: some of a state's rows lie over others", what);
    // states that share no memory with each other, nor have parents or lengths among them
    std::vector<const uint8_t*> at(d.n_states);
    uintptr_t all = (uintptr_t)d.bytes;
    for (int i = 0; i < d.n_states; ++i) {
        EXB_REQUIRE(states[i], "%s: null state", what);
        at[i] = static_cast<const uint8_t*>(states[i]);
        all |= reinterpret_cast<uintptr_t>(states[i]);
    }
    for (const Dim& x : dims) all |= (uintptr_t)x.stride;
    std::sort(at.begin(), at.end());
    const bool apart = side_by_side(dims, extent, at);
    for (int i = 0; i < d.n_states; ++i) {
        for (int j = i + 1; !apart && j < d.n_states && at[j] < at[i] + extent; ++j)
            EXB_REQUIRE(!meet(dims, 0, d.bytes, at[j] - at[i]), "%s: two states share memory", what);
        auto among = [&](const void* p, int64_t n) {
            const uint8_t* b = static_cast<const uint8_t*>(p);
            return p && b < at[i] + extent && b + n * 4 > at[i];
        };
        EXB_REQUIRE(!among(parents, d.sentences * d.beams) && !among(lengths, d.sentences), "%s: parents or lengths lie among a state's rows", what);
    }
    bits = all;
    return EXB_OK;
}

template <typename U>
int launch(const exb_ctx* ctx, const ReorderArgs& a, int beams, cudaStream_t st) {
    const int64_t columns = a.positions * a.bytes / (int64_t)sizeof(U) * a.sentences * a.n_states * a.outer;
    // Four CTAs an SM (64 states with 2 of 4 beams changed, 4, 6, 8 and 16: 42.1, 46.6, 43.8, 48.7 us).  Values on their way are registers: with 16 bytes each, four
    // columns of up to 4 beams, two of 8, one of more; smaller units take more columns (43 channels in fp32, 1, 2, 4 and 8 columns: 231, 98, 105, 78 us).
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
    for (int32_t i = 0; i < n; ++i) {
        uintptr_t bits;
        if (int rc = look_over("exb_reorder_beams_check", d[i], states[i], parents, lengths, bits)) return rc;
    }
    return EXB_OK;
} catch (const std::bad_alloc&) {
    return fail(EXB_ERR_NOMEM, "exb_reorder_beams_check: no memory for the list of states");
}

extern "C" int exb_reorder_beams_fwd(exb_ctx* ctx, const exb_reorder_desc* d, void* const* states, const int32_t* parents, const int32_t* lengths, void* stream) try {
    EXB_REQUIRE(ctx != nullptr && d != nullptr, "exb_reorder_beams_fwd: null context or descriptor");
    uintptr_t bits;
    if (int rc = look_over("exb_reorder_beams_fwd", *d, states, parents, lengths, bits)) return rc;
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
