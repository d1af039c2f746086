// Element types and pieces of rows for the row operators.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "row_ops.h"

namespace nvmai {

__device__ __forceinline__ float elem_to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float elem_to_float(float v) { return v; }
__device__ __forceinline__ float elem_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T elem_from_float(float v);
template <> __device__ __forceinline__ __half elem_from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float elem_from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 elem_from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// element i of an array whose type is known at run time only (routing weights, outputs of small calls)
__device__ __forceinline__ float load_elem(const void *p, uint32_t elem, size_t i) {
    if (elem == ELEM_F16) return __half2float(static_cast<const __half *>(p)[i]);
    if (elem == ELEM_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    return static_cast<const float *>(p)[i];
}

__device__ __forceinline__ void store_elem(void *p, uint32_t elem, size_t i, float v) {
    if (elem == ELEM_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else if (elem == ELEM_BF16) static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<float *>(p)[i] = v;
}

// V neighbouring elements, moved in one access (V * sizeof(T) <= 16 bytes, aligned to that)
template <typename T, int V> struct alignas(sizeof(T) * V) Piece { T v[V]; };

// ---- symmetric 8-bit codes of a row (nvmai_cuda_moe_quantize_rows) ----------------------------------------
// Every step is one rounding to fp32, so any order of the elements gives the same codes.  kTinyRow: below it 127 / m would
// overflow.  An infinite or NaN m: codes of 0 and a scale of NaN.
constexpr float kTinyRow = 7.52316385e-37f;      // 2^-120
struct RowScale { float scale, inverse; };
__device__ __forceinline__ RowScale row_scale(float m, bool finite) {
    RowScale r;
    r.scale = !finite ? __int_as_float(0x7fffffff) : m < kTinyRow ? 0.0f : __fdiv_rn(m, 127.0f);
    r.inverse = !finite || m < kTinyRow ? 0.0f : __fdiv_rn(127.0f, m);
    return r;
}
__device__ __forceinline__ int8_t row_code(float x, RowScale r) {
    return r.inverse == 0.0f ? (int8_t)0 : (int8_t)__float2int_rn(x * r.inverse);
}
// Largest magnitude so far, as a bit pattern: unsigned integers order like non-negative floats, with infinity and then the NaNs
// on top, so that one maximum also says whether everything is finite.
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ RowScale row_scale_bits(uint32_t m) { return row_scale(__uint_as_float(m), m < 0x7f800000u); }

}  // namespace nvmai
