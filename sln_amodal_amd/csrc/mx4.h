// Shared pieces of the microscaled 4-bit kernels (format: mx4.hip).
#pragma once
#include "mfma_nt.h"

#define MX_STEP 256              // a code row is padded to whole steps of 256 values (128 B)
#define MX_MAX_K (1 << 22)       // 128 rows of codes stay below 2^32 bytes

// Eight values from column k on; columns at or behind K are zero.  vec: rows start on 16-byte boundaries.
__device__ __forceinline__ void mx_load8(const float *row, int k, int K, int vec, float *v) {
    if (vec && k + 8 <= K) {
        const float4 a = *(const float4 *)(row + k), b = *(const float4 *)(row + k + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k + e < K ? row[k + e] : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void mx_load8(const T *row, int k, int K, int vec, float *v) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    if (vec && k + 8 <= K) {
        const t8 a = *(const t8 *)(row + k);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)a[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k + e < K ? (float)row[k + e] : 0.f;
    }
}
__device__ __forceinline__ void mx_store8(float *row, int k, int K, int vec, const float *v) {
    if (vec && k + 8 <= K) {
        *(float4 *)(row + k) = make_float4(v[0], v[1], v[2], v[3]);
        *(float4 *)(row + k + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < K) row[k + e] = v[e];
    }
}
template <typename T>
__device__ __forceinline__ void mx_store8(T *row, int k, int K, int vec, const float *v) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    if (vec && k + 8 <= K) {
        t8 a;
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = (T)v[e];
        *(t8 *)(row + k) = a;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < K) row[k + e] = (T)v[e];
    }
}

// Scale byte of block `blk` (32 values) of row `row` of R rows: [step][row][8], so that the scales of one 256-value step
// of neighbouring rows are neighbours (row-major they cost the product a cache line per row and step: 16000 x 12544 x
// 1024 took 198 us instead of 155).
__host__ __device__ __forceinline__ int64_t mx_scale_at(int64_t R, int64_t row, int blk) {
    return ((int64_t)(blk >> 3) * R + row) * 8 + (blk & 7);
}

// 2^(code - 127); code 0 is the subnormal 2^-127, 255 is NaN
__device__ __forceinline__ float mx_scale_value(unsigned code) {
    return __uint_as_float(code == 255u ? 0x7fc00000u : (code ? code << 23 : 0x00400000u));
}
// The values of eight codes (exact in float32)
__device__ __forceinline__ void mx_values8(unsigned q, unsigned scale_code, float *v) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const float s = mx_scale_value(scale_code);
    const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 1);
    const f2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 3);
    v[0] = a[0] * s; v[1] = a[1] * s; v[2] = b[0] * s; v[3] = b[1] * s;
    v[4] = c[0] * s; v[5] = c[1] * s; v[6] = d[0] * s; v[7] = d[1] * s;
}
