// 8-bit activation checkpoints: rows of 16/32-bit values to e4m3 with one power-of-two scale per 32 columns, and back
// (the form and its rounding: q8.h). Both are one pass over the data and bound by memory.
//
// Layout: a lane owns 8 consecutive columns, so 4 lanes share a group (two xor-shuffles give its amax); widths that
// are no multiple of 8 and strides or addresses off 16 bytes go element by element, 32 lanes a group.
// Median times (us, bf16): 16384 x 2736 25.5 to 8 bits (136 MB) and 21.6 back (part of them from the last-level cache);
// 16384 x 2731, element by element, 110 and 68: bound by the loads' and stores' count and the index's division, not by memory.
#include "q8.h"
#include "../../include/octsam.h"

namespace {
using namespace octsam;

// one lane: 8 columns of one row. nch = ceil(cols / 8) padded to a multiple of 4, so that the lanes of a group share
// a wave and run together
template <int TY>
__global__ __launch_bounds__(256) void quant8_vec_kernel(const void* __restrict__ x, long long ldx, long long rows,
                                                         int cols, int nch, uint8_t* __restrict__ q, long long ldq,
                                                         uint8_t* __restrict__ sc, long long lds_) {
  const long long total = rows * nch;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < ((total + 63) & ~63ll); i += (long long)gridDim.x * 256) {
    const long long r = i / nch;
    const int c = (int)(i - r * nch) * 8;
    const bool on = i < total && c < cols;
    float v[8];
    float m = 0.0f;
    if (on) {
      load8<TY>(x, r * ldx + c, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = q8_clean(v[e]);
        m = fmaxf(m, fabsf(v[e]));
      }
    }
    m = fmaxf(m, __shfl_xor(m, 1, 64));
    m = fmaxf(m, __shfl_xor(m, 2, 64));
    if (on) {
      const int b = q8_scale(m);
      const float inv = q8_inverse(b);
      *(u32x2*)(q + r * ldq + c) = (u32x2){q8_pack4(v, inv), q8_pack4(v + 4, inv)};
      if ((threadIdx.x & 3) == 0) sc[r * lds_ + (c >> 5)] = (uint8_t)b;
    }
  }
}

// any width, stride and alignment: a lane per column, 32 lanes per group
template <int TY>
__global__ __launch_bounds__(256) void quant8_any_kernel(const void* __restrict__ x, long long ldx, long long rows,
                                                         int cols, int ngr, uint8_t* __restrict__ q, long long ldq,
                                                         uint8_t* __restrict__ sc, long long lds_) {
  const int lane = threadIdx.x & 31;
  const long long total = rows * ngr;
  for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < ((total + 1) & ~1ll); i += (long long)gridDim.x * 8) {
    const long long r = i / ngr;
    const int g = (int)(i - r * ngr), c = g * 32 + lane;
    const bool on = i < total && c < cols;
    const float v = on ? q8_clean(load1<TY>(x, r * ldx + c)) : 0.0f;
    float m = fmaxf(0.0f, fabsf(v));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if (on) {
      const int b = q8_scale(m);
      q[r * ldq + c] = q8_pack1(v, q8_inverse(b));
      if (lane == 0) sc[r * lds_ + g] = (uint8_t)b;
    }
  }
}

template <int TY>
__global__ __launch_bounds__(256) void dequant8_vec_kernel(const uint8_t* __restrict__ q, long long ldq,
                                                           const uint8_t* __restrict__ sc, long long lds_, long long rows,
                                                           int cols, int nch, void* __restrict__ y, long long ldy) {
  const long long total = rows * nch;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long r = i / nch;
    const int c = (int)(i - r * nch) * 8;
    const u32x2 w = *(const u32x2*)(q + r * ldq + c);
    const float s = q8_value(sc[r * lds_ + (c >> 5)]);
    float v[8];
    q8_unpack4(w[0], s, v);
    q8_unpack4(w[1], s, v + 4);
    store8<TY>(y, r * ldy + c, v);
  }
}

template <int TY>
__global__ __launch_bounds__(256) void dequant8_any_kernel(const uint8_t* __restrict__ q, long long ldq,
                                                           const uint8_t* __restrict__ sc, long long lds_, long long rows,
                                                           int cols, void* __restrict__ y, long long ldy) {
  const long long total = rows * cols;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long r = i / cols;
    const int c = (int)(i - r * cols);
    store1<TY>(y, r * ldy + c, q8_unpack1(q[r * ldq + c], q8_value(sc[r * lds_ + (c >> 5)])));
  }
}

unsigned blocks_for(long long items, int per) {
  const long long n = (items + per - 1) / per;
  return (unsigned)(n < 16384 ? n : 16384);
}

}  // namespace

extern "C" int octsam_quant8(const void* x, int32_t x_type, int64_t ldx, int64_t rows, int32_t cols, void* q, int64_t ldq,
                             void* scale, int64_t ld_scale, void* stream) {
  OCTSAM_CHECK_ARG(type_ok(x_type), "quant8: x_type %d", x_type);
  OCTSAM_CHECK_ARG(rows >= 0 && cols >= 0 && rows <= (1ll << 40), "quant8: rows %lld, cols %d", (long long)rows, cols);
  if (rows == 0 || cols == 0) return 0;
  const int ngr = (int)(((int64_t)cols + 31) / 32);
  OCTSAM_CHECK_ARG(x && q && scale, "quant8: null operand");
  OCTSAM_CHECK_ARG(ldx >= cols && ldq >= cols && ld_scale >= ngr, "quant8: a row stride is below the row's width");
  OCTSAM_CHECK_ARG(aligned(x, type_size(x_type)), "quant8: x is not aligned to its type");
  const hipStream_t s = (hipStream_t)stream;
  const bool vec = cols % 8 == 0 && ldx % 8 == 0 && ldq % 8 == 0 && aligned(x, 16) && aligned(q, 8);
#define RUN(TY)                                                                                                         \
  if (vec)                                                                                                              \
    hipLaunchKernelGGL((quant8_vec_kernel<TY>), dim3(blocks_for(rows * (ngr * 4ll), 256)), dim3(256), 0, s, x, ldx, rows, \
                       cols, ngr * 4, (uint8_t*)q, ldq, (uint8_t*)scale, ld_scale);                                      \
  else                                                                                                                  \
    hipLaunchKernelGGL((quant8_any_kernel<TY>), dim3(blocks_for(rows * ngr, 8)), dim3(256), 0, s, x, ldx, rows, cols,    \
                       ngr, (uint8_t*)q, ldq, (uint8_t*)scale, ld_scale);
  if (x_type == T_BF16) { RUN(T_BF16) } else if (x_type == T_F32) { RUN(T_F32) } else { RUN(T_F16) }
#undef RUN
  OCTSAM_LAUNCH_CHECK("octsam_quant8");
  return 0;
}

extern "C" int octsam_dequant8(const void* q, int64_t ldq, const void* scale, int64_t ld_scale, int64_t rows, int32_t cols,
                               void* y, int32_t y_type, int64_t ldy, void* stream) {
  OCTSAM_CHECK_ARG(type_ok(y_type), "dequant8: y_type %d", y_type);
  OCTSAM_CHECK_ARG(rows >= 0 && cols >= 0 && rows <= (1ll << 40), "dequant8: rows %lld, cols %d", (long long)rows, cols);
  if (rows == 0 || cols == 0) return 0;
  const int ngr = (int)(((int64_t)cols + 31) / 32);
  OCTSAM_CHECK_ARG(y && q && scale, "dequant8: null operand");
  OCTSAM_CHECK_ARG(ldy >= cols && ldq >= cols && ld_scale >= ngr, "dequant8: a row stride is below the row's width");
  OCTSAM_CHECK_ARG(aligned(y, type_size(y_type)), "dequant8: y is not aligned to its type");
  const hipStream_t s = (hipStream_t)stream;
  const bool vec = cols % 8 == 0 && ldy % 8 == 0 && ldq % 8 == 0 && aligned(y, 16) && aligned(q, 8);
#define RUN(TY)                                                                                                        \
  if (vec)                                                                                                             \
    hipLaunchKernelGGL((dequant8_vec_kernel<TY>), dim3(blocks_for(rows * (cols / 8), 256)), dim3(256), 0, s,            \
                       (const uint8_t*)q, ldq, (const uint8_t*)scale, ld_scale, rows, cols, cols / 8, y, ldy);          \
  else                                                                                                                 \
    hipLaunchKernelGGL((dequant8_any_kernel<TY>), dim3(blocks_for(rows * cols, 256)), dim3(256), 0, s,                  \
                       (const uint8_t*)q, ldq, (const uint8_t*)scale, ld_scale, rows, cols, y, ldy);
  if (y_type == T_BF16) { RUN(T_BF16) } else if (y_type == T_F32) { RUN(T_F32) } else { RUN(T_F16) }
#undef RUN
  OCTSAM_LAUNCH_CHECK("octsam_dequant8");
  return 0;
}
