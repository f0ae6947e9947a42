// What the operators on rows of activations share: loads and stores of 8 elements of a row, the type dispatch, e4m3 blocks.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace exb {
namespace rows {

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }

// Two packed 16-bit elements as fp32.
__device__ __forceinline__ float2 pair_to_float(uint32_t v, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ float2 pair_to_float(uint32_t v, __nv_bfloat16) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
__device__ __forceinline__ uint32_t float_to_pair(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t float_to_pair(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// A warp's share of a row is 256 consecutive elements.  `valid`: elements of the row from the share's first one on (<= 0: none).
// How the lanes have them:
//  kVectors: 8 neighbours each, in 16-byte vectors: rows that start at multiples of 16 bytes and are whole vectors long;
//  kShifted: 8 neighbours each of rows that start anywhere, read in whole vectors and moved between lanes;
//  kStrided: every 32nd, loaded and stored one by one (64 or 128 bytes an instruction): rows that start anywhere.
enum Layout { kVectors, kShifted, kStrided };

// fp32 parameters of the share's channels.
template <Layout kL>
__device__ __forceinline__ void load8_params(const float* at, int valid, int lane, float2 (&v)[4]) {
    if constexpr (kL == kVectors) {
        if (lane * 8 < valid) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(at + lane * 8)), b = __ldg(reinterpret_cast<const float4*>(at + lane * 8) + 1);
            v[0] = make_float2(a.x, a.y);
            v[1] = make_float2(a.z, a.w);
            v[2] = make_float2(b.x, b.y);
            v[3] = make_float2(b.z, b.w);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = make_float2(0.f, 0.f);
        }
    } else {
        auto one = [&](int j) { return j * 32 + lane < valid ? __ldg(at + j * 32 + lane) : 0.f; };
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = make_float2(one(2 * j), one(2 * j + 1));
    }
}

// The memory that a tensor's rows may be read in: from its first element to behind its last row's last one.
struct Span {
    const uint8_t *begin, *end;
};
inline Span span_of(const void* p, int64_t rows, int64_t stride, int64_t C, size_t es) {
    const uint8_t* b = static_cast<const uint8_t*>(p);
    return {b, p ? b + ((rows - 1) * stride + C) * (int64_t)es : b};
}

// 16 bytes at a multiple of 16, or what of them lies in the span (elements of 2 or 4 bytes, whole).
template <int kBytes>
__device__ __forceinline__ uint4 load16_within(const uint8_t* at, const Span& span) {
    if (at >= span.begin && at + 16 <= span.end) return __ldg(reinterpret_cast<const uint4*>(at));
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 16; j += kBytes) {
        const uint8_t* e = at + j;
        if (e >= span.begin && e + kBytes <= span.end)
            w[j / 4] |= kBytes == 4 ? *reinterpret_cast<const uint32_t*>(e) : (uint32_t)*reinterpret_cast<const uint16_t*>(e) << (8 * (j & 2));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A warp's share of 256 elements, 8 neighbours in each lane, of a row that starts anywhere: whole 16-byte vectors are read, at
// multiples of 16 (fetch), and then moved into place between neighbouring lanes (settle).  Two steps, so that several rows can be
// asked for before the first is there.  Eight loads of single elements for each lane's 8 took three and a half times as long as aligned rows
// (8192 x 14335 bf16 to e4m3: 200 us; 56 aligned, 86 this way), both steps at once for each row 110 us.
// inside: no 16 bytes that hold some of the row reach out of the span (rows that have 8 others before and behind them).
template <typename T>
__device__ __forceinline__ void fetch8_shifted(const T* row_at, int valid, int lane, const Span& span, bool inside, uint32_t (&x)[2 * sizeof(T) + 4]) {
    constexpr int kWords = 2 * sizeof(T), kVecs = kWords / 4;          // of a lane
    const uintptr_t a = reinterpret_cast<uintptr_t>(row_at);
    const int o = (int)(a & 15);
    const uint8_t* base = reinterpret_cast<const uint8_t*>(a - o);
    const int bytes = o + min(valid, 256) * (int)sizeof(T);            // needed from base on
#pragma unroll
    for (int i = 0; i <= kVecs; ++i) {      // (what follows the last lane's own vectors, it reads itself)
        const int at = (lane * kVecs + i) * 16;
        uint4 q = make_uint4(0, 0, 0, 0);
        if (at < bytes && (i < kVecs || lane == 31)) q = inside ? __ldg(reinterpret_cast<const uint4*>(base + at)) : load16_within<sizeof(T)>(base + at, span);
        x[4 * i] = q.x; x[4 * i + 1] = q.y; x[4 * i + 2] = q.z; x[4 * i + 3] = q.w;
    }
}
template <typename T>
__device__ __forceinline__ void settle8_shifted(const T* row_at, int valid, int lane, uint32_t (&x)[2 * sizeof(T) + 4]) {
    constexpr int kWords = 2 * sizeof(T);
    const int o = (int)(reinterpret_cast<uintptr_t>(row_at) & 15);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t next = __shfl_down_sync(0xffffffffu, x[i], 1);
        if (lane < 31) x[kWords + i] = next;
    }
    // by o bytes: two words, one word, half a word
    if (o & 8) {
#pragma unroll
        for (int i = 0; i < kWords + 2; ++i) x[i] = x[i + 2];
    }
    if (o & 4) {
#pragma unroll
        for (int i = 0; i < kWords + 1; ++i) x[i] = x[i + 1];
    }
    if constexpr (sizeof(T) == 2) {
        const int sh = (o & 2) * 8;
#pragma unroll
        for (int i = 0; i < kWords; ++i) x[i] = __funnelshift_r(x[i], x[i + 1], sh);
    }
    // behind the row's end: 0
    constexpr int kPer = 4 / sizeof(T);
    if (lane * 8 + 8 > valid) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const int left = valid - lane * 8 - i * kPer;
            if (left <= 0) x[i] = 0;
            else if (kPer == 2 && left == 1) x[i] &= 0xffffu;
        }
    }
}

// A lane's 8 elements, kept as they are in memory until they are needed: 4 registers for 16-bit elements that are neighbours.
template <typename T, Layout kL>
struct Kept {
    static constexpr bool kPacked = sizeof(T) == 2 && kL != kStrided;
    static constexpr int kWords = kPacked ? 4 : 8;
    uint32_t w[kWords + (kL == kShifted ? 4 : 0)];
    __device__ __forceinline__ void none() {
#pragma unroll
        for (uint32_t& v : w) v = 0;
    }
    __device__ __forceinline__ void load(const T* at, int valid, int lane, const Span& span = {}, bool inside = false) {
        if constexpr (kL == kVectors) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                uint4 q = make_uint4(0, 0, 0, 0);
                if (lane * 8 < valid) q = reinterpret_cast<const uint4*>(at + lane * 8)[i];
                w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
            }
        } else if constexpr (kL == kShifted) {
            fetch8_shifted<T>(at, valid, lane, span, inside, w);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = j * 32 + lane < valid ? __float_as_uint(to_float<T>(at[j * 32 + lane])) : 0u;
        }
    }
    // (for rows that start anywhere, before anything is taken; by the whole warp)
    __device__ __forceinline__ void settle(const T* at, int valid, int lane) {
        if constexpr (kL == kShifted) settle8_shifted<T>(at, valid, lane, w);
    }
    __device__ __forceinline__ void get(float2 (&o)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (kPacked) o[i] = pair_to_float(w[i], T());
            else o[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        }
    }
    // the largest magnitude; NaN are left out
    __device__ __forceinline__ float amax() const {
        if constexpr (kPacked) {
            using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
            auto part = [&](int i) { return __habs2(*reinterpret_cast<const T2*>(&w[i])); };
            const T2 m = __hmax2(__hmax2(part(0), part(1)), __hmax2(part(2), part(3)));
            const float2 f = pair_to_float(*reinterpret_cast<const uint32_t*>(&m), T());
            return fmaxf(f.x, f.y);
        } else {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(__uint_as_float(w[i])));
            return m;
        }
    }
};

template <typename T, Layout kL>
__device__ __forceinline__ void store8(T* at, int valid, int lane, const float2 (&v)[4]) {
    static_assert(kL != kShifted, "results are written in vectors or one by one");
    if constexpr (kL == kVectors) {
        if (lane * 8 < valid) {
            if constexpr (sizeof(T) == 4) {
                float4* dst = reinterpret_cast<float4*>(at + lane * 8);
                dst[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
                dst[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
            } else {
                *reinterpret_cast<uint4*>(at + lane * 8) = make_uint4(float_to_pair(v[0].x, v[0].y, T()), float_to_pair(v[1].x, v[1].y, T()),
                                                                      float_to_pair(v[2].x, v[2].y, T()), float_to_pair(v[3].x, v[3].y, T()));
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (2 * j * 32 + lane < valid) at[2 * j * 32 + lane] = from_float<T>(v[j].x);
            if ((2 * j + 1) * 32 + lane < valid) at[(2 * j + 1) * 32 + lane] = from_float<T>(v[j].y);
        }
    }
}

// ---- e4m3 blocks of 128 --------------------------------------------------------------------
constexpr int kBlock = 128;
constexpr float kE4m3Max = 448.f;
// The smallest normal number: a block of zeros has it too, so that no scale is 0 and every reciprocal is finite.
constexpr float kSmallestScale = 1.17549435e-38f;

__device__ __forceinline__ float block_scale(float amax) { return fmaxf(amax / kE4m3Max, kSmallestScale); }
__device__ __forceinline__ uint32_t to_e4m3x4(float2 a, float2 b) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3), hi = __nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3);
    return __byte_perm(lo, hi, 0x5410);
}
__device__ __forceinline__ uint8_t to_e4m3(float a) { return (uint8_t)__nv_cvt_float_to_fp8(a, __NV_SATFINITE, __NV_E4M3); }

// 8 neighbours, of which `valid` are the row's.
__device__ __forceinline__ void store8_e4m3(uint8_t* q, const float2 (&v)[4], float inv, int valid) {
    const float2 ii = make_float2(inv, inv);
    const uint32_t lo = to_e4m3x4(__fmul2_rn(v[0], ii), __fmul2_rn(v[1], ii)), hi = to_e4m3x4(__fmul2_rn(v[2], ii), __fmul2_rn(v[3], ii));
    if (valid >= 8) {
        *reinterpret_cast<uint2*>(q) = make_uint2(lo, hi);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < valid) q[j] = (uint8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
    }
}

// kN values of each lane, kN a power of two up to 16: the largest of value number lane % kN over the 16 lanes of a block.  Each step
// hands half of the values to the neighbour that keeps them, so that 4 values take 5 exchanges instead of 16.  fmaxf drops NaN.
template <int kN>
__device__ __forceinline__ float largest_of_block(float (&m)[kN], int lane) {
    int step = 1;
#pragma unroll
    for (int n = kN; n > 1; n /= 2, step *= 2) {
        const bool odd = (lane & step) != 0;
#pragma unroll
        for (int j = 0; j < n / 2; ++j) {
            const float keep = odd ? m[2 * j + 1] : m[2 * j], give = odd ? m[2 * j] : m[2 * j + 1];
            m[j] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, give, step));
        }
    }
    for (; step < 16; step *= 2) m[0] = fmaxf(m[0], __shfl_xor_sync(0xffffffffu, m[0], step));
    return m[0];
}

// kN shares (two blocks of 128 each, 16 lanes a block, 8 neighbours a lane) -> e4m3 and their blocks' scales.  m: each lane's largest
// magnitudes; a block's scale comes from its numbers, a NaN itself goes into q.  A scale costs two IEEE divisions, 40 instructions
// where a share's 8 elements cost 60: lane i works out that of share i % kN, for all lanes of its block.
// values(i, v): the lane's elements of share i; q_at(i, valid): where it goes and how many elements it has (0: none); scale_at(i): where its first block's scale goes.
template <int kN, typename V, typename Q, typename S>
__device__ __forceinline__ void quantize_shares(V&& values, float (&m)[kN], int lane, int64_t scale_stride, Q&& q_at, S&& scale_at) {
    const float s = block_scale(largest_of_block<kN>(m, lane)), inv = 1.f / s;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        int valid;      // of the share's elements
        uint8_t* q = q_at(i, valid);
        const float each = __shfl_sync(0xffffffffu, inv, (lane & 16) + i);
        float2 v[4];
        values(i, v);
        if (lane * 8 < valid) store8_e4m3(q + lane * 8, v, each, valid - lane * 8);
        if ((lane & 15) == i && (lane >> 4) * kBlock < valid) scale_at(i)[(lane >> 4) * scale_stride] = s;
    }
}
// The same of every 32nd element: a lane has four of each block.
__device__ __forceinline__ void quantize8_strided(const float2 (&v)[4], int valid, int lane, uint8_t* __restrict__ q, float* __restrict__ scale,
                                                  int64_t scale_stride) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const float u[4] = {v[2 * b].x, v[2 * b].y, v[2 * b + 1].x, v[2 * b + 1].y};
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) m = fmaxf(m, fabsf(u[j]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float s = block_scale(m), inv = 1.f / s;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (b * kBlock + j * 32 + lane < valid) q[b * kBlock + j * 32 + lane] = to_e4m3(u[j] * inv);
        if (lane == 0 && b * kBlock < valid) scale[b * scale_stride] = s;
    }
}
__device__ __forceinline__ float largest_of(const float2 (&v)[4]) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = fmaxf(m, fmaxf(fabsf(v[j].x), fabsf(v[j].y)));
    return m;
}

// ---- host ----------------------------------------------------------------------------------
inline size_t element_size(int dtype) { return dtype == EXB_F32 ? 4 : dtype == EXB_F16 || dtype == EXB_BF16 ? 2 : 0; }
inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
// Whether rows at this base and stride can be read in 16-byte vectors (a missing tensor can).
inline bool vector_rows(const void* p, int64_t stride, size_t es) { return !p || (aligned16(p) && stride * (int64_t)es % 16 == 0); }

// Where a matrix lies: `rows` times `width` bytes, `stride` bytes apart (a missing tensor: no rows).
struct Place {
    const uint8_t* at;
    int64_t rows, width, stride;
};
inline Place place_of(const void* p, int64_t rows, int64_t C, int64_t stride, size_t es) {
    // (a single row's distance to the next means nothing)
    return {static_cast<const uint8_t*>(p), p ? rows : 0, C * (int64_t)es, (rows > 1 ? stride : C) * (int64_t)es};
}
inline bool same_place(const Place& a, const Place& b) { return a.at == b.at && a.rows == b.rows && a.width == b.width && a.stride == b.stride; }

// Whether two matrices share a byte.  Those that lie next to each other in the rows of a wider one do not.  Almost all calls are answered by
// the two ends or by equal strides; otherwise each row of the shorter one is looked for among the other's.
inline bool overlap(const Place& a, const Place& b) {
    if (a.rows == 0 || b.rows == 0) return false;
    auto end = [](const Place& p) { return p.at + (p.rows - 1) * p.stride + p.width; };
    if (a.at >= end(b) || b.at >= end(a)) return false;
    const Place &few = a.rows <= b.rows ? a : b, &many = a.rows <= b.rows ? b : a;
    // the last row of `many` that starts at `d` bytes from its first one or before
    auto before = [&](int64_t d) { return d >= 0 ? d / many.stride : -((-d + many.stride - 1) / many.stride); };
    const int64_t d = few.at - many.at;
    if (few.stride == many.stride) {      // row i of `few` lies m bytes behind row q + i of `many`
        const int64_t q = before(d), m = d - q * many.stride;
        auto both = [&](int64_t shift) { return shift < many.rows && shift + few.rows > 0; };
        return (m < many.width && both(q)) || (m + few.width > many.stride && both(q + 1));
    }
    for (int64_t i = 0; i < few.rows; ++i) {
        const int64_t at = d + i * few.stride;
        int64_t row = before(at + few.width - 1);
        if (row >= many.rows) row = many.rows - 1;
        if (row >= 0 && row * many.stride + many.width > at) return true;
    }
    return false;
}

// Whether one of the results shares a byte with an input or with another result.
template <int kOut, int kIn>
inline bool results_overlap(const Place (&out)[kOut], const Place (&in)[kIn]) {
    for (int i = 0; i < kOut; ++i) {
        for (const Place& p : in)
            if (overlap(out[i], p)) return true;
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], out[j])) return true;
    }
    return false;
}

// A launch goes to the calling thread's current device, whatever the context's and the addresses': on another one it would read memory that is
// not there.
inline int check_device(const exb_ctx* ctx, const char* what) {
    int device;
    EXB_CUDA_TRY(cudaGetDevice(&device));
    EXB_REQUIRE(device == ctx->device, "%s: the context is for device %d, the current device is %d", what, ctx->device, device);
    return EXB_OK;
}

// fn(T()) for the element type
template <typename F>
inline void with_type(int dtype, F&& fn) {
    if (dtype == EXB_F16) fn(__half());
    else if (dtype == EXB_BF16) fn(__nv_bfloat16());
    else fn(float());
}

}  // namespace rows
}  // namespace exb
