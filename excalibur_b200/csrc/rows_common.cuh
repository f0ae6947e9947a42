// What the operators on rows of activations share: loads and stores of 8 elements of a row, the type dispatch, e4m3 blocks.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

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

// A warp's share of a row is 256 consecutive elements, 8 of them in each lane: 8 neighbours in 16-byte vectors (kVec), or
// every 32nd in single elements where rows start anywhere (8 loads of 32 neighbours each: 64 bytes a load, which still
// is more than memory delivers).  `at`: the share's first element, `valid`: elements of the row from there on (<= 0: none).
// With kVec the row's length is a multiple of 8.
template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T* at, int valid, int lane, float (&v)[8]) {
    if constexpr (kVec) {
        if (lane * 8 < valid) {
            const uint4* src = reinterpret_cast<const uint4*>(at + lane * 8);
            if constexpr (sizeof(T) == 4) {
                const uint4 a = src[0], b = src[1];
                v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
                v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
            } else {
                const uint4 a = src[0];
                const float2 p0 = pair_to_float(a.x, T()), p1 = pair_to_float(a.y, T()), p2 = pair_to_float(a.z, T()), p3 = pair_to_float(a.w, T());
                v[0] = p0.x; v[1] = p0.y; v[2] = p1.x; v[3] = p1.y; v[4] = p2.x; v[5] = p2.y; v[6] = p3.x; v[7] = p3.y;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j * 32 + lane < valid ? to_float<T>(at[j * 32 + lane]) : 0.f;
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
// multiples of 16, and moved into place between neighbouring lanes.  About 20 instructions for 8 elements of 16 bits; eight loads
// of single elements for each lane's 8 took 3.7 times the time of aligned rows (8192 x 14335 bf16 to e4m3: 200 us, 63 aligned).
template <typename T>
__device__ __forceinline__ void load8_shifted(const T* row_at, int valid, int lane, const Span& span, float (&v)[8]) {
    constexpr int kWords = 8 * sizeof(T) / 4, kVecs = kWords / 4;      // of a lane
    const uintptr_t a = reinterpret_cast<uintptr_t>(row_at);
    const int o = (int)(a & 15);
    const uint8_t* base = reinterpret_cast<const uint8_t*>(a - o);
    const int bytes = o + min(valid, 256) * (int)sizeof(T);            // needed from base on
    uint32_t x[kWords + 4];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int at = (lane * kVecs + i) * 16;
        const uint4 q = at < bytes ? load16_within<sizeof(T)>(base + at, span) : make_uint4(0, 0, 0, 0);
        x[4 * i] = q.x; x[4 * i + 1] = q.y; x[4 * i + 2] = q.z; x[4 * i + 3] = q.w;
    }
    uint4 last = make_uint4(0, 0, 0, 0);
    if (lane == 31 && 32 * kVecs * 16 < bytes) last = load16_within<sizeof(T)>(base + 32 * kVecs * 16, span);
    x[kWords] = __shfl_down_sync(0xffffffffu, x[0], 1);
    x[kWords + 1] = __shfl_down_sync(0xffffffffu, x[1], 1);
    x[kWords + 2] = __shfl_down_sync(0xffffffffu, x[2], 1);
    x[kWords + 3] = __shfl_down_sync(0xffffffffu, x[3], 1);
    if (lane == 31) {
        x[kWords] = last.x; x[kWords + 1] = last.y; x[kWords + 2] = last.z; x[kWords + 3] = last.w;
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
        for (int i = 0; i < 4; ++i) {
            const float2 f = pair_to_float(__funnelshift_r(x[i], x[i + 1], sh), T());
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(x[i]);
    }
    if (lane * 8 + 8 > valid) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (lane * 8 + j >= valid) v[j] = 0.f;
    }
}

// The same, kept as it is in memory until it is needed: 4 registers for 8 elements of 16 bits in vectors.
template <typename T, bool kVec>
struct Kept {
    static constexpr bool kPacked = kVec && sizeof(T) == 2;
    uint4 packed;
    float v[kPacked ? 1 : 8];
    __device__ __forceinline__ void load(const T* at, int valid, int lane) {
        if constexpr (kPacked) {
            packed = make_uint4(0, 0, 0, 0);
            if (lane * 8 < valid) packed = *reinterpret_cast<const uint4*>(at + lane * 8);
        } else {
            load8<T, kVec>(at, valid, lane, v);
        }
    }
    __device__ __forceinline__ void get(float (&o)[8]) const {
        if constexpr (kPacked) {
            const float2 a = pair_to_float(packed.x, T()), b = pair_to_float(packed.y, T()), c = pair_to_float(packed.z, T()), d = pair_to_float(packed.w, T());
            o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y; o[4] = c.x; o[5] = c.y; o[6] = d.x; o[7] = d.y;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = v[j];
        }
    }
};

template <typename T, bool kVec>
__device__ __forceinline__ void store8(T* at, int valid, int lane, const float (&v)[8]) {
    if constexpr (kVec) {
        if (lane * 8 < valid) {
            uint4* dst = reinterpret_cast<uint4*>(at + lane * 8);
            if constexpr (sizeof(T) == 4) {
                dst[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
                dst[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
            } else {
                dst[0] = make_uint4(float_to_pair(v[0], v[1], T()), float_to_pair(v[2], v[3], T()), float_to_pair(v[4], v[5], T()),
                                    float_to_pair(v[6], v[7], T()));
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j * 32 + lane < valid) at[j * 32 + lane] = from_float<T>(v[j]);
    }
}

// ---- e4m3 blocks of 128 --------------------------------------------------------------------
constexpr int kBlock = 128;
constexpr float kE4m3Max = 448.f;
// The smallest normal number: a block of zeros has it too, so that no scale is 0 and every reciprocal is finite.
constexpr float kSmallestScale = 1.17549435e-38f;

__device__ __forceinline__ float block_scale(float amax) { return fmaxf(amax / kE4m3Max, kSmallestScale); }
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint8_t to_e4m3(float a) { return (uint8_t)__nv_cvt_float_to_fp8(a, __NV_SATFINITE, __NV_E4M3); }

// 8 neighbours, of which `valid` are the row's.
__device__ __forceinline__ void store8_e4m3(uint8_t* q, const float (&v)[8], float inv, int valid) {
    const uint32_t lo = to_e4m3x2(v[0] * inv, v[1] * inv) | to_e4m3x2(v[2] * inv, v[3] * inv) << 16;
    const uint32_t hi = to_e4m3x2(v[4] * inv, v[5] * inv) | to_e4m3x2(v[6] * inv, v[7] * inv) << 16;
    if (valid >= 8) {
        *reinterpret_cast<uint2*>(q) = make_uint2(lo, hi);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < valid) q[j] = (uint8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
    }
}

// The warp's share (two blocks of 128) of a row -> e4m3 and its blocks' scales.  fmaxf drops NaN: a block's scale comes from
// its other values, the NaN itself goes into q.  kVec: 8 neighbours in each lane, else every 32nd.
template <bool kVec>
__device__ __forceinline__ void quantize8(const float (&v)[8], int valid, int lane, uint8_t* __restrict__ q, float* __restrict__ scale,
                                          int64_t scale_stride) {
    if constexpr (kVec) {      // 16 lanes have a block
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float s = block_scale(m), inv = 1.f / s;
        if (lane * 8 < valid) {
            store8_e4m3(q + lane * 8, v, inv, valid - lane * 8);
            if ((lane & 15) == 0) scale[(lane >> 4) * scale_stride] = s;
        }
    } else {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            float m = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) m = fmaxf(m, fabsf(v[4 * b + j]));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float s = block_scale(m), inv = 1.f / s;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (b * kBlock + j * 32 + lane < valid) q[b * kBlock + j * 32 + lane] = to_e4m3(v[4 * b + j] * inv);
            if (lane == 0 && b * kBlock < valid) scale[b * scale_stride] = s;
        }
    }
}

// ---- host ----------------------------------------------------------------------------------
inline size_t element_size(int dtype) { return dtype == EXB_F32 ? 4 : dtype == EXB_F16 || dtype == EXB_BF16 ? 2 : 0; }
inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
// Whether rows at this base and stride can be read in 16-byte vectors (a missing tensor can).
inline bool vector_rows(const void* p, int64_t stride, size_t es) { return !p || (aligned16(p) && stride * (int64_t)es % 16 == 0); }

// fn(T()) for the element type
template <typename F>
inline void with_type(int dtype, F&& fn) {
    if (dtype == EXB_F16) fn(__half());
    else if (dtype == EXB_BF16) fn(__nv_bfloat16());
    else fn(float());
}

}  // namespace rows
}  // namespace exb
