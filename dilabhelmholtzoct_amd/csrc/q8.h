// The library's 8-bit form of activations, and 16/32-bit element access by type.
//
// A row of C values is stored as C e4m3 bytes (OCP: 4 exponent bits, 3 fraction bits, largest value 448) and
// ceil(C / 32) scale bytes: byte b stands for 2^(b - 127) (e8m0; 255 is NaN) and multiplies the 32 consecutive
// columns of its group (the last group of a row may be shorter). Writing: amax = the largest finite |x| of the
// group, b = the smallest with amax <= 448 * 2^(b - 127), at least 1; the byte of x is x * 2^(127 - b) rounded to
// nearest even, NaN (0x7f) where x is not finite. A power of two costs nothing against amax / 448: the product with
// it is exact, so the only error is e4m3's half step (2^-4 relative; values below 2^-14 of the group's largest fall
// into e4m3's subnormals), and reading back is exact in bf16 too.
#pragma once
#include "common.h"

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2v __attribute__((ext_vector_type(2)));

namespace octsam {

constexpr int Q8_GROUP = 32;
// element types of the C ABI's *_type arguments
constexpr int T_BF16 = 0, T_F32 = 1, T_F16 = 2;
__host__ __device__ constexpr int type_size(int t) { return t == T_F32 ? 4 : 2; }

__device__ __forceinline__ int q8_scale(float amax) {  // amax finite, >= 0
  const uint32_t u = __builtin_bit_cast(uint32_t, amax);
  const int b = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
  return b < 1 ? 1 : b;
}
__device__ __forceinline__ float q8_inverse(int b) { return __builtin_bit_cast(float, (uint32_t)(254 - b) << 23); }
__device__ __forceinline__ float q8_value(int b) {  // 2^(b - 127), b in [0, 255]
  const uint32_t u = b == 0 ? 0x00400000u : b == 255 ? 0x7fc00000u : (uint32_t)b << 23;
  return __builtin_bit_cast(float, u);
}
// x, or NaN where it is not finite (inf * 0): what the functions below take. Maxima ignore NaN, products and the
// conversion keep it
__device__ __forceinline__ float q8_clean(float x) { return fmaf(x, 0.0f, x); }
__device__ __forceinline__ uint32_t q8_pack4(const float* x, float inv) {
  int r = 0;
  r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, r, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, r, true);
  return (uint32_t)r;
}
__device__ __forceinline__ uint8_t q8_pack1(float x, float inv) {
  return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(x * inv, 0.0f, 0, false) & 0xff);
}
__device__ __forceinline__ void q8_unpack4(uint32_t q, float s, float* x) {
  const f32x2v a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
  x[0] = a[0] * s;
  x[1] = a[1] * s;
  x[2] = b[0] * s;
  x[3] = b[1] * s;
}
__device__ __forceinline__ float q8_unpack1(uint8_t q, float s) {
  return __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false)[0] * s;
}

template <int TY>
struct Elem;
template <> struct Elem<T_BF16> { typedef bf16 t; typedef bf16x8 v8; };
template <> struct Elem<T_F16> { typedef f16 t; typedef f16x8 v8; };
template <> struct Elem<T_F32> { typedef float t; };

// 8 consecutive elements (16-B aligned) as fp32 / from fp32, rounded to nearest even once
template <int TY>
__device__ __forceinline__ void load8(const void* base, long long i, float* v) {
  if constexpr (TY == T_F32) {
    const f32x4 a = *(const f32x4*)((const float*)base + i), b = *(const f32x4*)((const float*)base + i + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = a[e];
      v[4 + e] = b[e];
    }
  } else {
    const auto a = *(const typename Elem<TY>::v8*)((const typename Elem<TY>::t*)base + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)a[e];
  }
}
template <int TY>
__device__ __forceinline__ void store8(void* base, long long i, const float* v) {
  if constexpr (TY == T_F32) {
    *(f32x4*)((float*)base + i) = (f32x4){v[0], v[1], v[2], v[3]};
    *(f32x4*)((float*)base + i + 4) = (f32x4){v[4], v[5], v[6], v[7]};
  } else {
    typename Elem<TY>::v8 a;
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = (typename Elem<TY>::t)v[e];
    *(typename Elem<TY>::v8*)((typename Elem<TY>::t*)base + i) = a;
  }
}
template <int TY>
__device__ __forceinline__ float load1(const void* base, long long i) { return (float)((const typename Elem<TY>::t*)base)[i]; }
template <int TY>
__device__ __forceinline__ void store1(void* base, long long i, float v) {
  ((typename Elem<TY>::t*)base)[i] = (typename Elem<TY>::t)v;
}

inline bool type_ok(int t) { return t >= 0 && t <= 2; }
inline bool aligned(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

// Column sums of `rows` fp32 rows in fixed order by a workgroup of 256: SUM_COLS columns from c0 on, sixteen rows at a time
// (many loads in flight: the sum is a chain of latencies otherwise).
constexpr int SUM_COLS = 16;
__device__ __forceinline__ void column_sums(const float* __restrict__ part, int rows, int cols, int c0, float* __restrict__ out) {
  __shared__ float fold[16][SUM_COLS];
  const int lane = threadIdx.x & 15, sub = threadIdx.x >> 4, c = c0 + lane;
  float t = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int k = sub; k < rows; k += 16) t += part[(long long)k * cols + c];
  }
  fold[sub][lane] = t;
  __syncthreads();
  if (sub == 0 && c < cols) {
#pragma unroll
    for (int k = 1; k < 16; ++k) t += fold[k][lane];
    out[c] = t;
  }
}

}  // namespace octsam
