// Log probabilities of given tokens, the entropy and the most probable tokens of rows of logits.
//
// z = scale * x, p = exp(z - lse), lse = log sum exp z.  With any e, t = x * scale * log2(e) - e, s = sum 2^t, w = sum 2^t * t:
//   log p(v) = ln 2 * (t_v - log2 s),  entropy = ln 2 * (log2 s - w / s).
// One pass over the row, bound by its reading and, in 16 bits, by the latency of its loads (46 to 49 % of the issue slots are used, 40 to
// 46 % of the warps' stalls are waits for logits, and a CTA's loads drain at its row's end): 2048 rows of 50001 fp16 take 46.2 us with the
// top 5 (4430 GB/s), 40.7 without, 54.7 with 20; 1024 rows of 50000 fp32 without 36.4 (5630 GB/s); one row of 131072 fp32 with 20 7.9.
// A thread keeps an integer e near the largest value that it has seen, so that x * scale * log2(e) - e is one multiply-add with one
// rounding and a change of e scales its sums by a power of two, exactly.
//
// The most probable tokens come out of the same pass: a thread also keeps its largest logit.  The top-th largest of these (of groups
// of 8 threads in a CTA) is a lower bound tau of the answer, and only threads whose largest is not below tau hold anything
// that is not: about as many as tokens are asked for.  Their elements are read again (out of L2), those from tau on are put in
// order by counting for each how many are before it.  Logits and indexes make keys that are all different.  Where there are too many
// elements of equal value from tau on (masks, constant rows), the threads find out where their largest is, and the same
// is done with keys.
//
// A row that the pass cannot answer (a NaN or plus infinity in it, nothing but masks or logits at the type's lowest end, or more
// elements from tau on than there is room for) is answered by slow_row: the maximum, the sums about it, and one pass per token.
#include "ptx_sm100.cuh"
#include "rows_common.cuh"

namespace exb {
namespace {

using namespace rows;

constexpr int kMaxTop = 32;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct LogprobArgs {
    const void* logits;
    const int32_t* tokens;
    float *logprobs, *entropy, *top_logprobs;
    int32_t* top_tokens;
    int64_t stride;
    int V, n_given, top, splits;
    float scale;
};

// Logits in an order of unsigned numbers: both zeros alike, all NaN alike and above infinity.  With the index behind it (the lower one
// is the larger key) no two keys are alike, and none is 0 or all ones: a search may start from either.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return x != x ? 0xfffffffeu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long key_of(float x, int index) { return (unsigned long long)order_of(x) << 32 | (uint32_t)~index; }

__device__ __forceinline__ float logit_of(unsigned long long key) {      // (not of a NaN)
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int index_of(unsigned long long key) { return (int)~(uint32_t)key; }

__device__ __forceinline__ float exp2_fast(float t) {
    float p;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(t));
    return p;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// A 16-byte vector of logits: the largest of its parts (NaN if one is) kept packed, its elements, and these no lower than kLow (minus
// infinity would make 0 * infinity of p * t).
template <typename T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int kCount = 4;
    static constexpr float kLow = -1e30f;
    typedef float Max;
    static __device__ __forceinline__ Max largest(const uint4& v) {
        return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
    }
    static __device__ __forceinline__ Max larger(Max a, Max b) { return max_nan(a, b); }
    static __device__ __forceinline__ float value(Max m) { return m; }
    static __device__ __forceinline__ void elements(const uint4& v, float2 (&x)[2]) {
        x[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
        x[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
    }
    static __device__ __forceinline__ void bounded(const uint4& v, float2 (&x)[2]) {
        elements(v, x);
#pragma unroll
        for (int j = 0; j < 2; ++j) x[j] = make_float2(fmaxf(x[j].x, kLow), fmaxf(x[j].y, kLow));
    }
};
template <typename T, typename T2>
struct Vec16 {
    static constexpr int kCount = 8;
    typedef T2 Max;
    static __device__ __forceinline__ T2 part(uint32_t v) { return *reinterpret_cast<const T2*>(&v); }
    static __device__ __forceinline__ Max largest(const uint4& v) {
        return __hmax2_nan(__hmax2_nan(part(v.x), part(v.y)), __hmax2_nan(part(v.z), part(v.w)));
    }
    static __device__ __forceinline__ Max larger(Max a, Max b) { return __hmax2_nan(a, b); }
    static __device__ __forceinline__ float value(Max m) {
        const float2 f = pair_to_float(*reinterpret_cast<const uint32_t*>(&m), T());
        return max_nan(f.x, f.y);
    }
    static __device__ __forceinline__ void elements(const uint4& v, float2 (&x)[4]) {
        x[0] = pair_to_float(v.x, T());
        x[1] = pair_to_float(v.y, T());
        x[2] = pair_to_float(v.z, T());
        x[3] = pair_to_float(v.w, T());
    }
    static __device__ __forceinline__ void bounded_by(const uint4& v, uint32_t low, float2 (&x)[4]) {
        const T2 l = part(low);
        const T2 a = __hmax2(part(v.x), l), b = __hmax2(part(v.y), l), c = __hmax2(part(v.z), l), d = __hmax2(part(v.w), l);
        elements(make_uint4(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b), *reinterpret_cast<const uint32_t*>(&c),
                            *reinterpret_cast<const uint32_t*>(&d)), x);
    }
};
template <>
struct Vec<__half> : Vec16<__half, __half2> {
    static constexpr float kLow = -65504.f;
    static __device__ __forceinline__ void bounded(const uint4& v, float2 (&x)[4]) { bounded_by(v, 0xfbfffbffu, x); }
};
template <>
struct Vec<__nv_bfloat16> : Vec16<__nv_bfloat16, __nv_bfloat162> {
    static constexpr float kLow = -9.9e29f;      // (0xf149 is lower)
    static __device__ __forceinline__ void bounded(const uint4& v, float2 (&x)[4]) { bounded_by(v, 0xf149f149u, x); }
};

// Sums about a thread's (or a row's) reference e, and its largest logit (NaN if there is one).
struct alignas(16) Sums {
    float e, s, w, m;
};

// The lanes' sums joined, alike in all lanes (a sum over pairs does not depend on their order).  A lane without anything has e = -inf.
__device__ __forceinline__ Sums warp_sums(const Sums& a) {
    Sums r = a;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        r.e = fmaxf(r.e, __shfl_xor_sync(0xffffffffu, r.e, o));
        r.m = max_nan(r.m, __shfl_xor_sync(0xffffffffu, r.m, o));
    }
    const float d = a.e == r.e ? 0.f : fmaxf(a.e - r.e, -1000.f), f = exp2_fast(d);      // (not the difference of two infinities)
    r.s = a.s * f;
    r.w = fmaf(d, a.s, a.w) * f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
        r.w += __shfl_xor_sync(0xffffffffu, r.w, o);
    }
    return r;
}

// Where a row's whole 16-byte vectors are, and the single elements before (head) and behind them (tail).
template <typename T>
struct Parts {
    int head, vecs, tail0;
    const uint4* body;
    __device__ __forceinline__ Parts(const T* x, int V) {
        head = min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T), V);
        vecs = (V - head) / Vec<T>::kCount;
        tail0 = head + vecs * Vec<T>::kCount;
        body = reinterpret_cast<const uint4*>(x + head);
    }
};

// A thread's share of a row: every `step`-th of the vectors from `first` below `end`, and an element of the head and of the tail at most.
template <typename T>
struct Seen {
    // vectors that are asked for at a time (16 bits: 4, 6 and 8 took 47.8, 47.1 and 49.8 us for 2048 rows of 50001)
    static constexpr int kAhead = sizeof(T) == 4 ? 8 : 6;
    Sums r = {-INFINITY, 0.f, 0.f, -INFINITY};
    float2 s2 = {0.f, 0.f}, w2 = {0.f, 0.f};      // on top of r.s and r.w
    float c;

    __device__ __forceinline__ void fold() {
        r.s += s2.x + s2.y;
        r.w += w2.x + w2.y;
        s2 = w2 = make_float2(0.f, 0.f);
    }
    // the sums about another e: v is far above it (in most rows only the first vectors are)
    __device__ __forceinline__ void rise(float v) {
        fold();
        if (v != v) {
            r.s = NAN;
            return;
        }
        if (v <= Vec<T>::kLow) return;      // masks by a low value are masks: a reference down there would overflow what is taken for kLow
        const float e = ceilf(v * c);
        if (r.e != -INFINITY) {
            const float d = fmaxf(r.e - e, -1000.f), f = exp2_fast(d);      // (0 from there on; d * s has to stay a number)
            r.w = (r.w + d * r.s) * f;
            r.s *= f;
        }
        r.e = e;
    }
    __device__ __forceinline__ void single(float v) {
        r.m = max_nan(r.m, v);
        if (!(v * c <= r.e + 4.f)) rise(v);
        if (r.e != -INFINITY) {
            const float t = fmaxf(fmaf(v, c, -r.e), -200.f), p = exp2_fast(t);
            r.s += p;
            r.w = fmaf(p, t, r.w);
        }
    }
    // n of the vectors are there
    __device__ __forceinline__ void vectors(const uint4 (&q)[kAhead], int n) {
        typename Vec<T>::Max m = Vec<T>::largest(q[0]);
#pragma unroll
        for (int j = 1; j < kAhead; ++j)
            if (j < n) m = Vec<T>::larger(m, Vec<T>::largest(q[j]));
        const float top = Vec<T>::value(m);
        r.m = max_nan(r.m, top);
        if (!(top * c <= r.e + 4.f)) rise(top);
        if (r.e == -INFINITY) return;      // nothing but masks so far
        const float2 cc = make_float2(c, c), ee = make_float2(-r.e, -r.e);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (j >= n) break;
            constexpr int kPairs = Vec<T>::kCount / 2;
            float2 x[kPairs];
            Vec<T>::bounded(q[j], x);
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                const float2 t = __ffma2_rn(x[k], cc, ee), p = make_float2(exp2_fast(t.x), exp2_fast(t.y));
                s2 = __fadd2_rn(s2, p);
                w2 = __ffma2_rn(p, t, w2);
            }
        }
    }
    __device__ __forceinline__ void stream(const uint4* body, int first, int end, int step) {
        int i = first;
        for (; i + (kAhead - 1) * step < end; i += kAhead * step) {
            uint4 q[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) q[j] = __ldg(body + i + j * step);
            vectors(q, kAhead);
        }
        if (i < end) {
            uint4 q[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (i + j * step < end) q[j] = __ldg(body + i + j * step);
            vectors(q, (end - i + step - 1) / step);
        }
        fold();
    }
};

// Key of a thread's largest logit (the first of equal ones); 0 where it has none.
template <typename T>
__device__ __noinline__ unsigned long long best_key(const T* x, const Parts<T>& part, int thread, int n_head, int n_tail, int first, int end, int step) {
    unsigned long long best = 0;
    auto look = [&](float v, int index) {
        const unsigned long long k = key_of(v, index);
        best = k > best ? k : best;
    };
    if (thread < n_head) look(to_float<T>(x[thread]), thread);
    for (int i = first; i < end; i += step) {
        float2 v[Vec<T>::kCount / 2];
        Vec<T>::elements(__ldg(part.body + i), v);
#pragma unroll
        for (int k = 0; k < Vec<T>::kCount / 2; ++k) {
            look(v[k].x, part.head + i * Vec<T>::kCount + 2 * k);
            look(v[k].y, part.head + i * Vec<T>::kCount + 2 * k + 1);
        }
    }
    if (thread < n_tail) look(to_float<T>(x[part.tail0 + thread]), part.tail0 + thread);
    return best;
}

// The keys from tau on among a thread's elements go to the list, `lanes` lanes reading its vectors together.
template <typename T>
__device__ __forceinline__ void collect(const T* x, const Parts<T>& part, unsigned long long tau, int thread, int n_head, int n_tail, int first, int end, int step,
                                        int lane, int lanes, unsigned long long* list, int* n_list, int room) {
    const float low = tau >> 32 ? logit_of(tau) : -INFINITY;
    auto offer = [&](float v, int index) {
        if (!(v >= low)) return;
        const unsigned long long k = key_of(v, index);
        if (k >= tau) {
            const int n = atomicAdd(n_list, 1);
            if (n < room) list[n] = k;
        }
    };
    if (lane == 0 && thread < n_head) offer(to_float<T>(x[thread]), thread);
    for (int i = first + lane * step; i < end; i += lanes * step) {
        const uint4 q = __ldg(part.body + i);
        if (!(Vec<T>::value(Vec<T>::largest(q)) >= low)) continue;
        float2 v[Vec<T>::kCount / 2];
        Vec<T>::elements(q, v);
#pragma unroll
        for (int k = 0; k < Vec<T>::kCount / 2; ++k) {
            offer(v[k].x, part.head + i * Vec<T>::kCount + 2 * k);
            offer(v[k].y, part.head + i * Vec<T>::kCount + 2 * k + 1);
        }
    }
    if (lane == 0 && thread < n_tail) offer(to_float<T>(x[part.tail0 + thread]), part.tail0 + thread);
}

// The n-th largest (1..32) of the lanes' values (0: none); 0 if there are fewer.  Each lane counts the larger ones, in 32 exchanges that
// need not wait for each other; the n-th is the smallest of those with fewer than n.
__device__ __forceinline__ uint32_t nth_largest(uint32_t v, int n) {
    int larger = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) larger += __shfl_sync(0xffffffffu, v, j) > v;
    return __reduce_min_sync(0xffffffffu, larger < n ? v : 0xffffffffu);
}

// How many of n keys are before (above) one.
__device__ __forceinline__ int count_before(const unsigned long long* keys, int n, unsigned long long key) {
    int before = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) before += keys[j] > key;
    return before;
}

constexpr int kSplitMax = 8;      // CTAs of kWide threads that share a row
constexpr int kWide = 512, kNarrow = 256;
constexpr int kRoom = 512;        // elements from tau on that are put in order

template <int kThreads>
struct Shared {
    Sums part[kThreads / 32];
    Sums row[kSplitMax];                                   // (of the cluster's CTAs, in the first one)
    unsigned long long best[kSplitMax * kMaxTop];         // the same: the `top` best of each, in order
    uint32_t largest[kThreads / 8];                        // of 8 threads each
    unsigned long long list[kRoom > kThreads ? kRoom : kThreads];
    int threads[kThreads];
    unsigned long long tau;
    int n_list, n_threads, too_many[kSplitMax];
    float part_f[kThreads / 32];
};

// Barriers and reductions of the threads that work on a row: a CTA, or a warp (kThreads 32).
template <int kThreads>
__device__ __forceinline__ void sync() {
    if constexpr (kThreads == 32) __syncwarp();
    else __syncthreads();
}
template <int kThreads, typename F>
__device__ __forceinline__ float group_reduce(float v, float* s_part, F op) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    if constexpr (kThreads > 32) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
        __syncthreads();
        v = s_part[0];
        for (int i = 1; i < kThreads / 32; ++i) v = op(v, s_part[i]);
    }
    return v;
}

// What is written of a row whose sums are known: s and w about e, with the largest logit m.  The sum, its logarithm and the distance of
// m from e are rounded each for itself: where one token has nearly everything, that comes out up to 1.2e-7 beyond 0 more often than not, and the exponential
// of such a log probability above 1, so both are kept in their range.
struct Row {
    float m, log_s, entropy;      // log_s: log2 of the sum about m
    bool empty;
    float scale;
    __device__ __forceinline__ float logprob(float v) const {
        // (halves: the distance of fp32's two ends is no fp32 number)
        return empty ? -INFINITY : min_nan((0.5f * v - 0.5f * m) * (2.f * scale) - log_s * kLn2, 0.f);
    }
};

// Whether the pass has answered the row: its sums are numbers (the products in w are not where scaled logits lie further apart than fp32
// reaches), and what was taken for kLow has added nothing to them.
template <typename T>
__device__ __forceinline__ bool row_known(const Sums& all, float c) {
    return all.s > 0.f && all.s < INFINITY && fabsf(all.w) < INFINITY && fmaf(Vec<T>::kLow, c, -all.e) < -150.f;
}

template <typename T>
__device__ __forceinline__ void write_given(const LogprobArgs& a, const T* x, int64_t row, const Row& r, int first, int step) {
    for (int j = first; j < a.n_given; j += step) {
        const int token = a.tokens[row * a.n_given + j];
        a.logprobs[row * a.n_given + j] = token < 0 ? 0.f : token >= a.V ? NAN : r.logprob(to_float<T>(x[token]));
    }
}

template <typename T, int kThreads>
__device__ __noinline__ void slow_row(const LogprobArgs& a, const T* x, int64_t row, float* s_part, unsigned long long* s_best, bool sums_known, Row r) {
    const int tid = kThreads == 32 ? threadIdx.x & 31 : threadIdx.x;
    if (!sums_known) {
        const float c = a.scale * kLog2e;
        float m = -INFINITY, s = 0.f, w = 0.f;
        for (int i = tid; i < a.V; i += kThreads) m = fmaxf(m, to_float<T>(x[i]));
        m = group_reduce<kThreads>(m, s_part, [](float u, float v) { return fmaxf(u, v); });
        for (int i = tid; i < a.V; i += kThreads) {
            const float v = to_float<T>(x[i]), t = (v - m) * c, p = v == -INFINITY ? 0.f : exp2f(t);
            s += p;
            w += p == 0.f ? 0.f : p * t;
        }
        s = group_reduce<kThreads>(s, s_part, [](float u, float v) { return u + v; });
        w = group_reduce<kThreads>(w, s_part, [](float u, float v) { return u + v; });
        r.m = m;
        r.log_s = log2f(s);
        r.empty = !(s != 0.f);       // (a NaN anywhere makes s one)
        r.entropy = r.empty ? 0.f : (r.log_s - w / s) * kLn2;
        if (tid == 0 && a.entropy) a.entropy[row] = r.entropy;
        write_given<T>(a, x, row, r, tid, kThreads);
    }
    unsigned long long last = ~0ull;      // (above every key; top <= V, so that each pass finds one)
    for (int j = 0; j < a.top; ++j) {
        unsigned long long best = 0;
        for (int i = tid; i < a.V; i += kThreads) {
            const unsigned long long k = key_of(to_float<T>(x[i]), i);
            if (k < last && k > best) best = k;
        }
        sync<kThreads>();
        if (tid == 0) *s_best = 0;
        sync<kThreads>();
        atomicMax(s_best, best);
        sync<kThreads>();
        last = *static_cast<volatile unsigned long long*>(s_best);
        if (tid == 0) {
            const int token = index_of(last);
            a.top_tokens[row * a.top + j] = token;
            a.top_logprobs[row * a.top + j] = r.logprob(to_float<T>(x[token]));
        }
    }
}

// A warp's row each: short rows, whose exchange between warps would take longer than their reading.
// A lane has one largest logit, so that 32 alternatives reach down to the least of 32 maxima: 130 elements on the average, and more than 512 in
// one of 200 000 rows.  Rows of so few tokens that fewer lanes hold any than alternatives are asked for have 262 at most and are all
// candidates.  (With room for 128 both took a pass over the row for each alternative: 8192 rows of 1000 fp16 with 32 238 us, of 200 119.)
constexpr int kWarpRows = 4, kWarpRoom = 512;

// Of n keys those whose logit is not below the top-th largest, which is searched bit by bit; returns how many (more than `top` only for
// equal logits).  Counting for each key how many are before it takes n^2 / 32 steps of a warp: faster
// up to about 128 keys, but 72 us for 8192 rows with 200 (33 this way).
__device__ __forceinline__ int keep_largest(unsigned long long* keys, int n, int top, int lane) {
    uint32_t low = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t at = low | 1u << bit;
        int above = 0;
        for (int k = lane; k < n; k += 32) above += (uint32_t)(keys[k] >> 32) >= at;
        if ((int)__reduce_add_sync(0xffffffffu, above) >= top) low = at;
    }
    int kept = 0;
    for (int k0 = 0; k0 < n; k0 += 32) {      // (to the front: what is overwritten has been read)
        const unsigned long long key = k0 + lane < n ? keys[k0 + lane] : 0;
        const bool keep = key >> 32 >= low;      // (low is not 0: no key is)
        const uint32_t which = __ballot_sync(0xffffffffu, keep);
        if (keep) keys[kept + __popc(which & ((1u << lane) - 1))] = key;
        kept += __popc(which);
        __syncwarp();
    }
    return kept;
}

template <typename T>
__global__ void __launch_bounds__(kWarpRows * 32) token_logprobs_warp_kernel(const __grid_constant__ LogprobArgs a, int64_t n_rows) {
    __shared__ unsigned long long s_list[kWarpRows][kWarpRoom], s_best[kWarpRows];
    __shared__ int s_n[kWarpRows];
    pdl_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = (int64_t)blockIdx.x * kWarpRows + warp;
    if (row >= n_rows) return;
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    const Parts<T> part(x, a.V);
    const int n_tail = a.V - part.tail0;
    Seen<T> seen;
    seen.c = a.scale * kLog2e;
    if (lane < part.head) seen.single(to_float<T>(x[lane]));
    seen.stream(part.body, lane, part.vecs, 32);
    if (lane < n_tail) seen.single(to_float<T>(x[part.tail0 + lane]));
    const Sums all = warp_sums(seen.r);
    Row out;
    out.scale = a.scale;
    out.m = all.m;
    out.empty = false;
    const bool known = row_known<T>(all, seen.c);
    if (known) {
        const float log_s = log2f(all.s);
        out.entropy = max_nan((log_s - all.w / all.s) * kLn2, 0.f);
        out.log_s = log_s - fmaf(all.m, seen.c, -all.e);
        if (lane == 0 && a.entropy) a.entropy[row] = out.entropy;
        write_given<T>(a, x, row, out, lane, 32);
    }
    bool slow = !known;
    if (known && a.top) {
        const bool any = lane < part.head || lane < part.vecs || lane < n_tail;
        const uint32_t mine = any ? order_of(seen.r.m) : 0;
        unsigned long long tau = (unsigned long long)nth_largest(mine, a.top) << 32;
        bool looked = any && mine >= tau >> 32;
        int n;
        for (int tries = 0;; ++tries) {
            if (lane == 0) s_n[warp] = 0;
            __syncwarp();
            if (part.vecs <= 32 * 8) {      // each lane reads its own few vectors again, otherwise the warp one lane's after the other
                if (looked) collect<T>(x, part, tau, lane, part.head, n_tail, lane, part.vecs, 32, 0, 1, s_list[warp], &s_n[warp], kWarpRoom);
            } else {
                for (uint32_t left = __ballot_sync(0xffffffffu, looked); left; left &= left - 1) {
                    const int t = __ffs(left) - 1;
                    collect<T>(x, part, tau, t, part.head, n_tail, t, part.vecs, 32, lane, 32, s_list[warp], &s_n[warp], kWarpRoom);
                }
            }
            __syncwarp();
            n = *static_cast<volatile int*>(&s_n[warp]);
            __syncwarp();
            if (n <= kWarpRoom || tries) break;
            // too many of equal value: the same with keys
            const unsigned long long key = best_key<T>(x, part, lane, part.head, n_tail, lane, part.vecs, 32);
            unsigned long long left = key;
            tau = 0;
            for (int j = 0; j < a.top; ++j) {
                const uint32_t h = __reduce_max_sync(0xffffffffu, (uint32_t)(left >> 32)), l = __reduce_max_sync(0xffffffffu, (uint32_t)(left >> 32) == h ? (uint32_t)left : 0u);
                tau = (unsigned long long)h << 32 | l;
                if (left == tau) left = 0;
            }
            looked = key != 0 && key >= tau;
        }
        slow = n > kWarpRoom;
        if (n > 128 && !slow) n = keep_largest(s_list[warp], n, a.top, lane);
        for (int k = lane; k < n && !slow; k += 32) {
            const unsigned long long mine_ = s_list[warp][k];
            const int before = count_before(s_list[warp], n, mine_);
            if (before < a.top) {
                a.top_tokens[row * a.top + before] = index_of(mine_);
                a.top_logprobs[row * a.top + before] = out.logprob(logit_of(mine_));
            }
        }
    }
    if (slow) slow_row<T, 32>(a, x, row, nullptr, &s_best[warp], known, out);
}

// gridDim.x = rows * splits, the CTAs of a row are a cluster (kNarrow threads: one CTA a row).
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const __grid_constant__ LogprobArgs a) {
    __shared__ Shared<kThreads> sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int splits = kThreads == kWide ? a.splits : 1;
    const int64_t row = blockIdx.x / splits;
    const int rank = (int)(blockIdx.x - row * splits);
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    // Of the row's vectors this CTA has [lo, hi) and a thread every kThreads-th; the head is with the first CTA, the tail with the last.
    const Parts<T> part(x, a.V);
    const int head = part.head, vecs = part.vecs, tail0 = part.tail0;
    const uint4* body = part.body;
    const int lo = (int)((int64_t)rank * vecs / splits), hi = (int)((int64_t)(rank + 1) * vecs / splits);
    const int n_head = rank == 0 ? head : 0, n_tail = rank == splits - 1 ? a.V - tail0 : 0;
    const float c = a.scale * kLog2e;
    if (tid == 0) {
        sh.n_list = 0;
        sh.n_threads = 0;
        sh.tau = 0;
    }
    if (splits > 1) ptx::cluster_arrive();      // (waited for before anything is written into the first CTA)
    pdl_enter();

    Seen<T> seen;
    seen.c = c;
    if (tid < n_head) seen.single(to_float<T>(x[tid]));
    seen.stream(body, lo + tid, hi, kThreads);
    if (tid < n_tail) seen.single(to_float<T>(x[tail0 + tid]));

    Sums all = warp_sums(seen.r);
    if (lane == 0) sh.part[warp] = all;
    const bool any = tid < n_head || lo + tid < hi || tid < n_tail;
    const uint32_t mine = any ? order_of(seen.r.m) : 0;
    if (a.top) {
        uint32_t g = mine;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
        if ((lane & 7) == 0) sh.largest[tid >> 3] = g;
    }
    if (splits > 1) {
        __syncwarp();
        ptx::cluster_wait();
    }
    __syncthreads();
    bool too_many = false;
    int n_best = 0;
    if (a.top) {
        if (warp == 0) {      // (with 64 groups a lane has the larger of two: the bound is lower, and serves all the same)
            uint32_t g = sh.largest[lane];
            if constexpr (kThreads == kWide) g = max(g, sh.largest[lane + 32]);
            g = nth_largest(g, a.top);
            if (lane == 0) sh.tau = (unsigned long long)g << 32;
        }
        __syncthreads();
        unsigned long long tau = sh.tau;
        bool looked = any && mine >= tau >> 32;
        int n;
        for (int tries = 0;; ++tries) {
            if (looked) sh.threads[atomicAdd(&sh.n_threads, 1)] = tid;
            __syncthreads();
            const int n_threads = sh.n_threads;
            // (all threads for a bound that few tokens are above: masks)
            if (tries || n_threads <= kThreads / 2) {
                for (int w = warp; w < n_threads; w += kThreads / 32) {
                    const int t = sh.threads[w];
                    collect<T>(x, part, tau, t, n_head, n_tail, lo + t, hi, kThreads, lane, 32, sh.list, &sh.n_list, kRoom);
                }
                __syncthreads();
                n = sh.n_list;
            } else {
                n = kRoom + 1;
            }
            if (n <= kRoom || tries) break;
            // too many of equal value, or no bound: of up to 2048 16-bit tokens fewer than 32 groups of 8 threads hold any (256 x 1100 fp16 with
            // 5 alternatives 5.6 us, with 20, which come this way, 15.8).  The top-th largest of the threads' keys is one.
            const unsigned long long key = best_key<T>(x, part, tid, n_head, n_tail, lo + tid, hi, kThreads);
            __syncthreads();
            sh.list[tid] = key;
            if (tid == 0) {
                sh.n_threads = 0;
                sh.tau = 0;
            }
            __syncthreads();
            const int before = count_before(sh.list, kThreads, key);
            if (key && before == a.top - 1) sh.tau = key;
            __syncthreads();
            tau = sh.tau;
            looked = key != 0 && key >= tau;
            if (tid == 0) sh.n_list = 0;
        }
        too_many = n > kRoom;
        n_best = min(n, a.top);
        if (!too_many) {
            unsigned long long* to = splits > 1 ? nullptr : sh.best;
            for (int k = tid; k < n; k += kThreads) {
                const unsigned long long key = sh.list[k];
                const int before = count_before(sh.list, n, key);
                if (before < a.top) {
                    if (to) to[before] = key;
                    else ptx::st_cta_u64(ptx::map_to_cta(ptx::smem_u32(&sh.best[rank * a.top + before]), 0), key);
                }
            }
            if (splits > 1 && tid >= n_best && tid < a.top) ptx::st_cta_u64(ptx::map_to_cta(ptx::smem_u32(&sh.best[rank * a.top + tid]), 0), 0);
        }
    }
    // (the warps' sums, in every warp for itself)
    all = warp_sums(lane < kThreads / 32 ? sh.part[lane] : Sums{-INFINITY, 0.f, 0.f, -INFINITY});
    if (splits > 1) {      // the first CTA finishes the row
        if (tid == 0) {
            const uint32_t to = ptx::map_to_cta(ptx::smem_u32(&sh.row[rank]), 0);
            ptx::st_cta_u64(to, (unsigned long long)__float_as_uint(all.s) << 32 | __float_as_uint(all.e));
            ptx::st_cta_u64(to + 8, (unsigned long long)__float_as_uint(all.m) << 32 | __float_as_uint(all.w));
            ptx::st_cta_u32(ptx::map_to_cta(ptx::smem_u32(&sh.too_many[rank]), 0), too_many ? 1u : 0u);
        }
        __syncwarp();
        ptx::cluster_sync();
        if (rank) return;
        all = warp_sums(lane < splits ? sh.row[lane] : Sums{-INFINITY, 0.f, 0.f, -INFINITY});
        too_many = __any_sync(0xffffffffu, lane < splits && sh.too_many[lane] != 0);
    }
    Row out;
    out.scale = a.scale;
    out.m = all.m;
    out.empty = false;
    const bool known = row_known<T>(all, a.scale * kLog2e);
    if (known) {
        const float log_s = log2f(all.s);
        out.entropy = max_nan((log_s - all.w / all.s) * kLn2, 0.f);
        out.log_s = log_s - fmaf(all.m, c, -all.e);
        if (tid == 0 && a.entropy) a.entropy[row] = out.entropy;
        write_given<T>(a, x, row, out, tid, kThreads);
    }
    if (!known || (a.top && too_many)) {
        slow_row<T, kThreads>(a, x, row, sh.part_f, &sh.tau, known, out);
        return;
    }
    if (a.top) {
        if (splits == 1) __syncthreads();
        const int n = splits * a.top;
        for (int k = tid; k < n; k += kThreads) {
            const unsigned long long mine = sh.best[k];
            const int before = splits == 1 ? k : count_before(sh.best, n, mine);
            if (before < a.top && mine) {
                a.top_tokens[row * a.top + before] = index_of(mine);
                a.top_logprobs[row * a.top + before] = out.logprob(logit_of(mine));
            }
        }
    }
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
    const int64_t bytes = (int64_t)V * (int64_t)es;
    int rc = EXB_OK;
    // A warp for a row where a CTA's exchange between warps takes longer than the reading, and where there are rows for all warps.  (fp16,
    // top 5, us with a warp and with a CTA for a row.  64 rows of 200: 3.3 and 13.2, of 1000: 4.4 and 4.2, of 2000: 5.7 and 4.4, of 8000:
    // 8.1 and 5.3.  1184 rows of 2000: 11.1 and 10.2, of 4000: 14.3 and 11.0; 1776 of 2000: 7.6 and 14.5, of 8000: 13.7 and 17.3;
    // 8192 of 4000: 23.7 and 60; 2368 of 16000: 31.8 and 28.0.)
    if (bytes <= 2048 || (bytes <= 16384 && n_rows >= 12 * ctx->sm_count)) {
        rows::with_type(dtype, [&](auto t) {
            using T = decltype(t);
            launch_overlapped(ctx, token_logprobs_warp_kernel<T>, dim3((unsigned)((n_rows + kWarpRows - 1) / kWarpRows)), dim3(kWarpRows * 32), st, a, n_rows);
        });
        return after_launch("token_logprobs_warp_kernel");
    }
    // Two CTAs of 512 threads fill an SM, four of 256.  As long as all rows have their CTAs at once the wide ones are the faster (fp16, us
    // with 512 and 256: 148 rows of 50000 9.0 and 9.9, 296 of them 11.1 and 17.0, 296 of 8000 6.1 and 7.3, of 131072 18.7 and 32.1);
    // with more rows the narrow ones leave less of a last wave empty (444 of 16000: 11.8 and 9.9, 2048 of 50000: 64.6 and 45.7).
    const bool wide = bytes >= 16384 && n_rows <= 2 * ctx->sm_count;
    // Fewer rows than SMs are shared by the CTAs of a cluster as long as each has three vectors for a thread (in 1, 2, 4, 8 parts: one row of
    // 131072 9.6, 8.0, 6.9, 6.6; 32 of them 14.5, 12.0, 10.2, 11.1; 74 12.8, 10.5, 15.7, 19.3; one row of 20000 4.7, 5.4, 5.5, 5.9).
    a.splits = 1;
    while (wide && a.splits < kSplitMax && n_rows * a.splits * 2 <= ctx->sm_count && bytes >= (int64_t)a.splits * 2 * kWide * 48) a.splits *= 2;
    rows::with_type(dtype, [&](auto t) {
        using T = decltype(t);
        rc = wide ? launch<T, kWide>(ctx, a, n_rows, st) : launch<T, kNarrow>(ctx, a, n_rows, st);
    });
    return rc;
}
