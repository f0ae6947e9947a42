// What the matrix products of 8- and 16-bit operands share: K blocks of 128 bytes, the stores of their results, the order of tiles, tensor maps.
#pragma once
#include "ptx_sm100.cuh"
#include "rows_common.cuh"
#include "tensor_map.cuh"

namespace exb {
namespace product {

constexpr int kBlk = 128;                  // K block: bytes of a row in a stage
constexpr uint32_t kMaxSpins = 1u << 21;

// kTmemOrder: a kernel whose CTAs took TMEM while they wait for the previous kernel could take what CTAs of that one, started but not
// that far, still need, and both would wait for good.  So TMEM is taken behind griddepcontrol.wait, and the next kernel is let in
// (griddepcontrol.launch_dependents) only behind that.

__device__ __forceinline__ void store_one(void* y, int dtype, int64_t at, float v) {
    if (dtype == EXB_F16) static_cast<__half*>(y)[at] = __float2half_rn(v);
    else if (dtype == EXB_BF16) static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
    else static_cast<float*>(y)[at] = v;
}

// Four neighbouring channels of a row.
__device__ __forceinline__ void store_four(void* y, int y_dtype, int64_t y_stride, int N, bool vec, int m, int n, const float (&v)[4]) {
    const int64_t at = (int64_t)m * y_stride + n;
    if (vec && n + 4 <= N) {
        if (y_dtype == EXB_F32)
            *reinterpret_cast<float4*>(static_cast<float*>(y) + at) = make_float4(v[0], v[1], v[2], v[3]);
        else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(y) + at) =
                y_dtype == EXB_F16 ? make_uint2(rows::float_to_pair(v[0], v[1], __half()), rows::float_to_pair(v[2], v[3], __half()))
                                     : make_uint2(rows::float_to_pair(v[0], v[1], __nv_bfloat16()), rows::float_to_pair(v[2], v[3], __nv_bfloat16()));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < N) store_one(y, y_dtype, at + j, v[j]);
    }
}

// Results of 32 rows x up to 128 bytes per warp, in units of 16 bytes that are XOR-ed with the row: a thread writes its row's units
// and the warp reads whole rows, both without bank conflicts.
constexpr int kStageOut = 32 * 128;

// Columns [col, col + 2 * kPairs) of 32 rows from row0 on: sums in `acc` (a thread has a row), through shared memory to y in whole vectors.
template <typename T, int kPairs>
__device__ __forceinline__ void store_rows(const float2 (&acc)[kPairs], uint8_t* stage, T* y, int64_t y_stride, int row0, int col, int M, int N, bool vec,
                                           int lane) {
    constexpr int kPer = 16 / (int)sizeof(T);                                                   // columns in a unit,
    constexpr int kUnits = 2 * kPairs / kPer < 8 ? 2 * kPairs / kPer : 8, kCols = kUnits * kPer;      // units and columns in a pass
    constexpr int kRows = 32 / kUnits;                                                          // rows that the warp writes at a time
    const int sub = lane / kUnits, u = lane % kUnits;
    auto unit = [&](int r, int i) { return reinterpret_cast<uint4*>(stage + r * 128 + ((i ^ (r & 7)) << 4)); };
    auto element = [&](int r, int e) { return reinterpret_cast<const T*>(unit(r, e / kPer))[e % kPer]; };
#pragma unroll
    for (int c0 = 0; c0 < 2 * kPairs; c0 += kCols) {
        if (col + c0 >= N) break;
        const int left = N - col - c0;
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const float2* v = acc + (c0 + i * kPer) / 2;
            if constexpr (sizeof(T) == 4)
                *unit(lane, i) = make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
            else
                *unit(lane, i) = make_uint4(rows::float_to_pair(v[0].x, v[0].y, T()), rows::float_to_pair(v[1].x, v[1].y, T()),
                                            rows::float_to_pair(v[2].x, v[2].y, T()), rows::float_to_pair(v[3].x, v[3].y, T()));
        }
        __syncwarp();
        T* out = y + (int64_t)row0 * y_stride + col + c0;
        if (left < kCols) {
            for (int r = 0; r < 32 && row0 + r < M; ++r) {
#pragma unroll
                for (int c = lane; c < kCols; c += 32)
                    if (c < left) out[r * y_stride + c] = element(r, c);
            }
        } else if (vec) {
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int r = i * kRows + sub;
                if (row0 + r < M) *reinterpret_cast<uint4*>(out + r * y_stride + u * kPer) = *unit(r, u);
            }
        } else {
            // Rows that start anywhere: kUnits - 1 vectors at multiples of 16 bytes, put together of two units each, and 16 bytes before
            // and behind them element by element.  (fp16, 4048 x 7313 x 264 takes
            // 42.9 us, element by element 51.8, and 4048 x 7312 x 264 29: sectors that two passes write a part of each are the difference.)
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const int r = i * kRows + sub;
                if (row0 + r >= M) continue;
                T* to = out + r * y_stride;
                const int o = (int)((16 - (reinterpret_cast<uintptr_t>(to) & 15)) & 15);      // bytes before the first multiple of 16
                if (o == 0) {
                    *reinterpret_cast<uint4*>(to + u * kPer) = *unit(r, u);
                    continue;
                }
                if (u < kUnits - 1) {
                    const uint4 a = *unit(r, u), b = *unit(r, u + 1);
                    uint32_t x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                    if (o & 8) {
#pragma unroll
                        for (int k = 0; k < 6; ++k) x[k] = x[k + 2];
                    }
                    if (o & 4) {
#pragma unroll
                        for (int k = 0; k < 5; ++k) x[k] = x[k + 1];
                    }
                    const int sh = (o & 2) * 8;
                    *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(to) + o + u * 16) =
                        make_uint4(__funnelshift_r(x[0], x[1], sh), __funnelshift_r(x[1], x[2], sh), __funnelshift_r(x[2], x[3], sh), __funnelshift_r(x[3], x[4], sh));
                }
#pragma unroll
                for (int k = 0; k < kPer; k += kUnits)      // as many elements before the first vector and behind the last as a unit has
                    if (k + u < kPer) {
                        const int e = (k + u) * (int)sizeof(T) < o ? k + u : kCols - kPer + k + u;
                        to[e] = element(r, e);
                    }
            }
        }
        __syncwarp();
    }
}

// Tiles in an order in which those that run at the same time share rows of a and w: columns of 8 tiles, one after the other.
__device__ __forceinline__ void tile_at(int t, int m_tiles, int n_tiles, int& m, int& n) {
    const int group = t / (8 * n_tiles), first = group * 8, size = min(m_tiles - first, 8);
    const int r = t - group * 8 * n_tiles;
    n = r / size;
    m = first + r - n * size;
}

template <int kRegs> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }

// Rows of K bytes in boxes of 128 bytes x box_rows, 128-byte swizzle; zeros beyond the matrix.
inline int encode_rows(const char* what, CUtensorMap* map, const uint8_t* base, int64_t rows, int K, int64_t stride, int box_rows) {
    const auto fn = tensor_map_encoder();
    if (!fn) return fail(EXB_ERR_CUDA, "%s: the driver has no cuTensorMapEncodeTiled", what);
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
    cuuint32_t box[2] = {(cuuint32_t)kBlk, (cuuint32_t)box_rows}, step[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(EXB_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
    return EXB_OK;
}

}  // namespace product
}  // namespace exb
