// Log probabilities of given tokens, the entropy and the most probable tokens of rows of logits.
//
// z = scale * x, p = exp(z - lse), lse = log sum exp z.  With any e, t = x * scale * log2(e) - e, s = sum 2^t, w = sum 2^t * t:
//   log p(v) = ln 2 * (t_v - log2 s),  entropy = ln 2 * (log2 s - w / s).
// One pass over the row, bound by its reading.  A thread keeps an integer e near the largest value that it has seen, so that
// x * scale * log2(e) - e is one multiply-add with one rounding and a change of e scales its sums by a power of two, exactly.
//
// The most probable tokens come out of the same pass: a thread also keeps its largest logit and the vector that has it.  The top-th
// largest of these is a lower bound tau of the answer, and only the threads whose largest is not below tau can hold
// anything that is not: about as many as tokens are asked for.  Their elements are read again (out of L2), those from tau on
// are put in order by counting for each how many are before it.  Logits and indexes make keys that are all different, so that
// equal logits, masked ones among them, need nothing else.
//
// A row that the pass cannot answer (a NaN or plus infinity in it, nothing but masks of fp32's or bf16's lowest value, or more
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

// Logits in an order of unsigned numbers: both zeros alike, NaN above infinity.  With the index behind it (the lower one is the larger
// key) no two keys are alike.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
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

// The largest of a 16-byte vector of logits, NaN if one is.
__device__ __forceinline__ float largest(const uint4& v, float) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
}
__device__ __forceinline__ float largest(const uint4& v, __half) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
}
__device__ __forceinline__ float largest(const uint4& v, __nv_bfloat16) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
}
template <typename T>
__device__ __forceinline__ void elements(const uint4& v, float (&x)[16 / sizeof(T)]) {
    if constexpr (sizeof(T) == 4) {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    } else {
        const float2 a = pair_to_float(v.x, T()), b = pair_to_float(v.y, T()), c = pair_to_float(v.z, T()), d = pair_to_float(v.w, T());
        x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
    }
}

// Sums about a thread's (or a row's) reference e, and its largest logit.
struct alignas(16) Sums {
    float e, s, w, m;
};
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b) {
    // (a side without anything has s = w = 0 and e = -inf: its factor is 0, and the difference of two infinities is not taken)
    Sums r;
    r.e = fmaxf(a.e, b.e);
    r.m = fmaxf(a.m, b.m);
    const float da = a.e == r.e ? 0.f : fmaxf(a.e - r.e, -1000.f), db = b.e == r.e ? 0.f : fmaxf(b.e - r.e, -1000.f);
    const float fa = exp2_fast(da), fb = exp2_fast(db);
    r.s = a.s * fa + b.s * fb;
    r.w = (a.w + da * a.s) * fa + (b.w + db * b.s) * fb;
    return r;
}

constexpr int kSplitMax = 8;      // CTAs that share a row
constexpr int kRoom = 512;        // elements from tau on that are put in order

template <int kThreads>
struct Shared {
    Sums part[kThreads / 32];
    Sums row[kSplitMax];                                   // (of the cluster's CTAs, in the first one)
    unsigned long long best[kSplitMax][kMaxTop];           // the same: their best, in order
    unsigned long long group[kThreads / 8];
    unsigned long long list[kRoom > kThreads ? kRoom : kThreads];
    int threads[kThreads];
    unsigned long long tau;
    int n_list, n_threads, too_many[kSplitMax];
    float part_f[kThreads / 32];
};

template <int kThreads, typename F>
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

// What is written of a row whose sums are known: s and w about e, with the largest logit m.
struct Row {
    float m, log_s, entropy;      // log_s: log2 of the sum about m
    bool empty;
    float scale;
    __device__ __forceinline__ float logprob(float v) const {
        // (halves: the distance of fp32's two ends is no fp32 number)
        return empty ? -INFINITY : (0.5f * v - 0.5f * m) * (2.f * scale) - log_s * kLn2;
    }
};

template <typename T>
__device__ __forceinline__ void write_given(const LogprobArgs& a, const T* x, int64_t row, const Row& r, int first, int step) {
    for (int j = first; j < a.n_given; j += step) {
        const int token = a.tokens[row * a.n_given + j];
        a.logprobs[row * a.n_given + j] = token < 0 ? 0.f : token >= a.V ? NAN : r.logprob(to_float<T>(x[token]));
    }
}

template <typename T, int kThreads>
__device__ __noinline__ void slow_row(const LogprobArgs& a, const T* x, int64_t row, Shared<kThreads>& sh, bool sums_known, Row r) {
    if (!sums_known) {
        const float c = a.scale * kLog2e;
        float m = -INFINITY, s = 0.f, w = 0.f;
        for (int i = threadIdx.x; i < a.V; i += kThreads) m = fmaxf(m, to_float<T>(x[i]));
        m = block_reduce<kThreads>(m, sh.part_f, [](float u, float v) { return fmaxf(u, v); });
        for (int i = threadIdx.x; i < a.V; i += kThreads) {
            const float v = to_float<T>(x[i]), t = (v - m) * c, p = v == -INFINITY ? 0.f : exp2f(t);
            s += p;
            w += p == 0.f ? 0.f : p * t;
        }
        s = block_reduce<kThreads>(s, sh.part_f, [](float u, float v) { return u + v; });
        w = block_reduce<kThreads>(w, sh.part_f, [](float u, float v) { return u + v; });
        r.m = m;
        r.log_s = log2f(s);
        r.empty = !(s != 0.f);       // (a NaN anywhere makes s one)
        r.entropy = r.empty ? 0.f : (r.log_s - w / s) * kLn2;
        if (threadIdx.x == 0 && a.entropy) a.entropy[row] = r.entropy;
        write_given<T>(a, x, row, r, threadIdx.x, kThreads);
    }
    unsigned long long last = ~0ull;
    for (int j = 0; j < a.top; ++j) {
        unsigned long long best = 0;
        for (int i = threadIdx.x; i < a.V; i += kThreads) {
            const unsigned long long k = key_of(to_float<T>(x[i]), i);
            if (k < last && k > best) best = k;
        }
        __syncthreads();
        if (threadIdx.x == 0) sh.tau = 0;
        __syncthreads();
        atomicMax(&sh.tau, best);
        __syncthreads();
        last = sh.tau;
        if (threadIdx.x == 0) {
            const int token = index_of(last);
            a.top_tokens[row * a.top + j] = token;
            a.top_logprobs[row * a.top + j] = r.logprob(to_float<T>(x[token]));
        }
    }
}

// gridDim.x = rows * splits, the CTAs of a row are a cluster.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const __grid_constant__ LogprobArgs a) {
    constexpr int kVec = 16 / sizeof(T), kAhead = 4;
    __shared__ Shared<kThreads> sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / a.splits;
    const int rank = (int)(blockIdx.x - row * a.splits);
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    // Whole 16-byte vectors, of which this CTA has [lo, hi) and a thread every kThreads-th, and single elements before (head, with
    // the first CTA) and behind them (tail, with the last).
    const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T), a.V);
    const int vecs = (a.V - head) / kVec, tail0 = head + vecs * kVec;
    const int lo = (int)((int64_t)rank * vecs / a.splits), hi = (int)((int64_t)(rank + 1) * vecs / a.splits);
    const uint4* body = reinterpret_cast<const uint4*>(x + head);
    const int n_head = rank == 0 ? head : 0, n_tail = rank == a.splits - 1 ? a.V - tail0 : 0;
    const float c = a.scale * kLog2e;
    if (tid == 0) {
        sh.n_list = 0;
        sh.n_threads = 0;
        sh.tau = 0;
    }
    if (a.splits > 1) ptx::cluster_arrive();      // (waited for before anything is written into the first CTA)
    pdl_enter();

    Sums r = {-INFINITY, 0.f, 0.f, -INFINITY};
    int at = -1;      // where r.m is: vector at, or the head's element (-1) or the tail's (-2)
    bool any = false;
    // what a new largest logit means: whether e still serves
    auto rise = [&](float v, int where) {
        if (v != v) {
            r.s = NAN;
            return;
        }
        r.m = v;
        at = where;
        const float e = ceilf(v * c);
        if (e > r.e + 4.f) {
            if (r.e != -INFINITY) {
                const float d = r.e - e, f = exp2_fast(d);
                r.w = (r.w + d * r.s) * f;
                r.s *= f;
            }
            r.e = e;
        }
    };
    auto single = [&](float v, int where) {
        any = true;
        if (!(v <= r.m)) rise(v, where);
        if (r.m != -INFINITY) {
            const float t = fmaxf(fmaf(v, c, -r.e), -200.f), p = exp2_fast(t);
            r.s += p;
            r.w = fmaf(p, t, r.w);
        }
    };
    if (tid < n_head) single(to_float<T>(x[tid]), -1);
    f32x2 s2 = pack2(0.f, 0.f), w2 = s2;
    auto fold = [&]() {
        float u, v;
        unpack2(s2, u, v);
        r.s += u + v;
        unpack2(w2, u, v);
        r.w += u + v;
        s2 = w2 = pack2(0.f, 0.f);
    };
    auto vector = [&](const uint4& q, int where) {
        const float m = largest(q, T());
        if (!(m <= r.m)) {
            fold();
            rise(m, where);
        }
        if (r.m == -INFINITY) return;      // nothing but masks so far
        float v[kVec];
        elements<T>(q, v);
        const f32x2 cc = pack2(c, c), ee = pack2(-r.e, -r.e);
#pragma unroll
        for (int j = 0; j < kVec; j += 2) {
            float t0, t1;
            unpack2(fma2(pack2(v[j], v[j + 1]), cc, ee), t0, t1);
            t0 = fmaxf(t0, -200.f);      // (p is 0 there and p * t has to be)
            t1 = fmaxf(t1, -200.f);
            const f32x2 p = pack2(exp2_fast(t0), exp2_fast(t1));
            s2 = add2(s2, p);
            w2 = fma2(p, pack2(t0, t1), w2);
        }
    };
    int i = lo + tid;
    if (i < hi) {
        if (!any) at = i;
        any = true;
    }
    for (; i + (kAhead - 1) * kThreads < hi; i += kAhead * kThreads) {
        uint4 q[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) q[j] = __ldg(body + i + j * kThreads);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) vector(q[j], i + j * kThreads);
    }
    for (; i < hi; i += kThreads) vector(__ldg(body + i), i);
    fold();
    if (tid < n_tail) {
        if (!any) at = -2;
        single(to_float<T>(x[tail0 + tid]), -2);
    }

    // the block's sums, in a fixed order
    Sums all = r;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Sums other = {__shfl_xor_sync(0xffffffffu, all.e, o), __shfl_xor_sync(0xffffffffu, all.s, o), __shfl_xor_sync(0xffffffffu, all.w, o),
                            __shfl_xor_sync(0xffffffffu, all.m, o)};
        all = (lane & o) ? joined(other, all) : joined(all, other);
    }
    if (lane == 0) sh.part[warp] = all;

    if (a.splits > 1) {
        __syncwarp();
        ptx::cluster_wait();
    }
    bool too_many = false;
    int n_best = 0;
    if (a.top) {
        // The thread's largest as a key that is not above the true one (the vector's last index), and one that is not below it.
        const int first_index = at == -1 ? tid : at == -2 ? tail0 + tid : head + at * kVec;
        const unsigned long long low = any ? key_of(r.m, first_index + (at >= 0 ? kVec - 1 : 0)) : 0, high = any ? key_of(r.m, first_index) : 0;
        // the top-th largest of the largest of 8 threads each: a first bound, so that few keys remain
        unsigned long long g = low;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, g, o);
            g = other > g ? other : g;
        }
        if ((lane & 7) == 0) sh.group[tid >> 3] = g;
        __syncthreads();
        if (tid < kThreads / 8) {
            const unsigned long long mine = sh.group[tid];
            int before = 0;
#pragma unroll 8
            for (int j = 0; j < kThreads / 8; ++j) before += sh.group[j] > mine;
            if (mine && before == a.top - 1) sh.tau = mine;
        }
        __syncthreads();
        const unsigned long long tau1 = sh.tau;
        if (low && low >= tau1) sh.list[atomicAdd(&sh.n_list, 1)] = low;      // (no more than there are threads)
        __syncthreads();
        const int n1 = sh.n_list;
        for (int k = tid; k < n1; k += kThreads) {      // the bound itself: the top-th largest of the threads'
            const unsigned long long mine = sh.list[k];
            int before = 0;
            for (int j = 0; j < n1; ++j) before += sh.list[j] > mine;
            if (before == a.top - 1) sh.tau = mine;
        }
        __syncthreads();
        const unsigned long long tau = sh.tau;
        if (any && high >= tau) sh.threads[atomicAdd(&sh.n_threads, 1)] = tid;
        if (tid == 0) sh.n_list = 0;
        __syncthreads();
        auto offer = [&](float v, int index) {
            const unsigned long long k = key_of(v, index);
            if (k >= tau) {
                const int n = atomicAdd(&sh.n_list, 1);
                if (n < kRoom) sh.list[n] = k;
            }
        };
        for (int w = warp; w < sh.n_threads; w += kThreads / 32) {      // a warp reads one thread's elements again
            const int t = sh.threads[w];
            if (lane == 0 && t < n_head) offer(to_float<T>(x[t]), t);
            if (lane == 1 && t < n_tail) offer(to_float<T>(x[tail0 + t]), tail0 + t);
            for (int j = lo + t + lane * kThreads; j < hi; j += 32 * kThreads) {
                float v[kVec];
                elements<T>(__ldg(body + j), v);
#pragma unroll
                for (int k = 0; k < kVec; ++k) offer(v[k], head + j * kVec + k);
            }
        }
        __syncthreads();
        const int n = sh.n_list;
        too_many = n > kRoom;
        n_best = min(n, a.top);
        if (!too_many) {
            unsigned long long* to = a.splits > 1 ? nullptr : sh.best[0];
            for (int k = tid; k < n; k += kThreads) {
                const unsigned long long mine = sh.list[k];
                int before = 0;
                for (int j = 0; j < n; ++j) before += sh.list[j] > mine;
                if (before < a.top) {
                    if (to) to[before] = mine;
                    else ptx::st_cta_u64(ptx::map_to_cta(ptx::smem_u32(&sh.best[rank][before]), 0), mine);
                }
            }
            if (a.splits > 1 && tid >= n_best && tid < a.top) ptx::st_cta_u64(ptx::map_to_cta(ptx::smem_u32(&sh.best[rank][tid]), 0), 0);
        }
    }
    __syncthreads();
    all = sh.part[0];
    for (int w = 1; w < kThreads / 32; ++w) all = joined(all, sh.part[w]);
    if (a.splits > 1) {      // the first CTA finishes the row
        if (tid == 0) {
            const uint32_t to = ptx::map_to_cta(ptx::smem_u32(&sh.row[rank]), 0);
            ptx::st_cta_u64(to, (unsigned long long)__float_as_uint(all.s) << 32 | __float_as_uint(all.e));
            ptx::st_cta_u64(to + 8, (unsigned long long)__float_as_uint(all.m) << 32 | __float_as_uint(all.w));
            ptx::st_cta_u32(ptx::map_to_cta(ptx::smem_u32(&sh.too_many[rank]), 0), too_many ? 1u : 0u);
        }
        __syncwarp();
        ptx::cluster_sync();
        if (rank) return;
        all = sh.row[0];
        too_many = sh.too_many[0] != 0;
        for (int k = 1; k < a.splits; ++k) {
            all = joined(all, sh.row[k]);
            too_many = too_many || sh.too_many[k] != 0;
        }
    }
    Row out;
    out.scale = a.scale;
    out.m = all.m;
    out.empty = false;
    const bool known = all.s > 0.f && all.s < INFINITY;
    if (known) {
        const float log_s = log2f(all.s);
        out.entropy = (log_s - all.w / all.s) * kLn2;
        out.log_s = log_s - fmaf(all.m, c, -all.e);
        if (tid == 0 && a.entropy) a.entropy[row] = out.entropy;
        write_given<T>(a, x, row, out, tid, kThreads);
    }
    if (!known || (a.top && too_many)) {
        slow_row<T, kThreads>(a, x, row, sh, known, out);
        return;
    }
    if (a.top) {
        const int n = a.splits * a.top;
        for (int k = tid; k < n; k += kThreads) {
            const unsigned long long mine = sh.best[k / a.top][k % a.top];
            int before = 0;
            if (a.splits == 1) before = k;
            else
                for (int j = 0; j < a.splits; ++j)
                    for (int l = 0; l < a.top; ++l) before += sh.best[j][l] > mine;
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
    const int64_t bytes = (int64_t)V * (int64_t)es;
    const int threads = bytes <= 8192 ? 128 : bytes >= 131072 && n_rows <= ctx->sm_count ? 512 : 256;
    // a row is shared where there are too few of them, as long as each CTA has two vectors for a thread
    a.splits = 1;
    while (a.splits < kSplitMax && n_rows * a.splits * 2 <= 2 * ctx->sm_count && bytes >= (int64_t)a.splits * 2 * threads * 32) a.splits *= 2;
    int rc = EXB_OK;
    rows::with_type(dtype, [&](auto t) {
        using T = decltype(t);
        rc = threads == 128 ? launch<T, 128>(ctx, a, n_rows, st) : threads == 256 ? launch<T, 256>(ctx, a, n_rows, st) : launch<T, 512>(ctx, a, n_rows, st);
    });
    return rc;
}
