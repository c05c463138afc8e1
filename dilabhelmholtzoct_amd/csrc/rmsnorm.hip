// Root-mean-square norm with the residual's addition in front of it, forward and backward.
//
//   s = x + r;  rstd = (mean(s^2) + eps)^(-1/2);  y = s * rstd * w                   (y from the unrounded fp32 s)
//   n = s * rstd;  g = dy * w;  ds = dres + rstd * (g - n * mean(g * n));  dw = sum over rows of dy * n
//
// ds is the gradient of both x and r. All sums and statistics are fp32; every output is rounded once. y can be written
// as 16/32-bit values and, from the same registers, in the library's 8-bit form (q8.h); the backward reads s as it was
// stored, or from its 8-bit form.
//
// Both directions are one pass over the rows and bound by memory. A row is owned by T lanes (16 .. 256 by its width),
// lane j holding the columns 8 (j + T c) .. + 7 in registers between the statistics and the outputs, so every operand
// is read once in 16-B (fp32: 2 x 16-B) pieces and four neighbouring lanes hold an 8-bit group. The backward keeps
// dw's columns in registers over a workgroup's rows, adds its row groups through LDS and leaves one partial row per
// workgroup, which a second launch adds in fixed order (results do not vary from run to run). Lanes past the row's end
// load its first columns and drop them, so that no branch stands between one load and the next. Widths that are no
// multiple of 8 and strides and addresses off 16 bytes take the same kernels with single elements (W = 1: lane j holds
// the columns j + T i, 32 lanes an 8-bit group). Rows over 8192 columns go column by column with a wave per row and are
// read twice.
//
// Median times (us, bf16, residual, the chip kept busy): forward of 16384 x 1024 21.8 (134 MB, part of them still in the
// last-level cache), with the 8-bit form 25.5; of 16384 x 1021 (single elements) 27.0, with the 8-bit form 46.3: there
// the maxima over 32 lanes and single bytes are the time. Backward of 16384 x 1280 34.3 (168 MB) and 4.7 for dw; of
// 16384 x 1021 26.7 from 16 bits (1024: 24.4), but 74 from 8 bits (1024: 22.8), a byte and its scale's byte a load.
#include "q8.h"
#include "../../include/octsam.h"

namespace {
using namespace octsam;
constexpr int T_NONE = -1, T_Q8 = 3;

struct NormFwd {
  const void *x, *r;
  const float* w;
  void *s, *y;
  uint8_t *q, *sc;
  float* rstd;
  long long ldx, ldr, lds, ldy, ldq, ldsc, rows;
  int D, y_type;
  float eps;
};

// a lane's elements of its row: NCH chunks of 8, element e of chunk c at column col_of(c, e). W = 8: 8 consecutive
// columns, all inside the row or all outside; W = 1: every element by itself
template <int T, int W>
__device__ __forceinline__ int col_of(int lane, int c, int e) { return W == 8 ? 8 * (lane + T * c) + e : lane + T * (8 * c + e); }
template <int TY, int T, int W>
__device__ __forceinline__ void load_chunk(const void* p, long long at, int lane, int c, int D, float* v) {
  if constexpr (W == 8) {
    const int col = col_of<T, W>(lane, c, 0);
    load8<TY>(p, at + (col < D ? col : 0), v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int col = col_of<T, W>(lane, c, e);
      v[e] = load1<TY>(p, at + (col < D ? col : 0));
    }
  }
}
// zeros in the place of columns past the row's end (D = 0: all)
template <int T, int W>
__device__ __forceinline__ void cut_chunk(int lane, int c, int D, float* v) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = col_of<T, W>(lane, c, e) < D ? v[e] : 0.0f;
}
template <int TY, int T, int W>
__device__ __forceinline__ void store_chunk(void* p, long long at, int lane, int c, int D, const float* v) {
  if constexpr (W == 8) {
    const int col = col_of<T, W>(lane, c, 0);
    if (col < D) store8<TY>(p, at + col, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int col = col_of<T, W>(lane, c, e);
      if (col < D) store1<TY>(p, at + col, v[e]);
    }
  }
}
template <int T, int W>
__device__ __forceinline__ void store_chunk_by(int type, void* p, long long at, int lane, int c, int D, const float* v) {
  if (type == T_BF16) store_chunk<T_BF16, T, W>(p, at, lane, c, D, v);
  else if (type == T_F32) store_chunk<T_F32, T, W>(p, at, lane, c, D, v);
  else store_chunk<T_F16, T, W>(p, at, lane, c, D, v);
}

template <int T>
__device__ __forceinline__ float group_total(float v, float* red) {
#pragma unroll
  for (int o = (T < 64 ? T : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (T > 64) {  // one row per workgroup
    __syncthreads();       // (red's readers of the row before)
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) v += red[i];
  }
  return v;
}

// v^(-1/2). 1 / sqrtf rounds twice, and a row's error goes into all of its values; a Newton step with the residue in two
// parts takes it to about half a step (not where v is 0 or infinite)
__device__ __forceinline__ float inverse_root(float v) {
  const float r = 1.0f / sqrtf(v), h = v * r;
  const float e = fmaf(-h, r, 1.0f) - fmaf(v, r, -h) * r;  // 1 - v r^2
  return fabsf(e) < 1e-3f ? fmaf(0.5f * r, e, r) : r;
}

__device__ __forceinline__ void store1_by(int type, void* p, long long i, float v) {
  if (type == T_BF16) store1<T_BF16>(p, i, v);
  else if (type == T_F32) store1<T_F32>(p, i, v);
  else store1<T_F16>(p, i, v);
}

template <int XT, int RT, int T, int NCH, int W>
__global__ __launch_bounds__(256) void rmsnorm_fwd_kernel(NormFwd a) {
  constexpr int RPB = 256 / T;
  __shared__ float red[4];
  const int lane = threadIdx.x % T;
  const float inv_d = 1.0f / (float)a.D;
  float w[NCH][8];
#pragma unroll
  for (int c = 0; c < NCH; ++c) load_chunk<T_F32, T, W>(a.w, 0, lane, c, a.D, w[c]);
  const long long last = (a.rows + RPB - 1) / RPB * RPB;  // (all lanes of a wave run every pass: they reduce together)
  for (long long row = (long long)blockIdx.x * RPB + threadIdx.x / T; row < last; row += (long long)gridDim.x * RPB) {
    const int D = row < a.rows ? a.D : 0;  // (a row past the end has no columns; it loads the last row's)
    const long long from = row < a.rows ? row : a.rows - 1;
    float v[NCH][8], r[RT != T_NONE ? NCH : 1][8];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      load_chunk<XT, T, W>(a.x, from * a.ldx, lane, c, a.D, v[c]);
      if constexpr (RT != T_NONE) load_chunk<RT, T, W>(a.r, from * a.ldr, lane, c, a.D, r[c]);
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if constexpr (RT != T_NONE) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] += r[c][e];
        if (a.s) store_chunk<RT, T, W>(a.s, row * a.lds, lane, c, D, v[c]);
      }
      cut_chunk<T, W>(lane, c, D, v[c]);
    }
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(v[c][e], v[c][e], ss);
    ss = group_total<T>(ss, red);
    const float rstd = inverse_root(fmaf(ss, inv_d, a.eps));
    if (D && lane == 0 && a.rstd) a.rstd[row] = rstd;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = v[c][e] * rstd * w[c][e];
      cut_chunk<T, W>(lane, c, D, v[c]);
      if (a.y) store_chunk_by<T, W>(a.y_type, a.y, row * a.ldy, lane, c, D, v[c]);
      if (a.q) {  // (uniform)
        if constexpr (W == 8) {
          float m = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[c][e] = q8_clean(v[c][e]);
            m = fmaxf(m, fabsf(v[c][e]));
          }
          m = fmaxf(m, __shfl_xor(m, 1, 64));
          m = fmaxf(m, __shfl_xor(m, 2, 64));
          const int col = col_of<T, W>(lane, c, 0);
          if (col < D) {
            const int b = q8_scale(m);
            const float inv = q8_inverse(b);
            *(u32x2*)(a.q + row * a.ldq + col) = (u32x2){q8_pack4(v[c], inv), q8_pack4(v[c] + 4, inv)};
            if ((lane & 3) == 0) a.sc[row * a.ldsc + (col >> 5)] = (uint8_t)b;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float y = q8_clean(v[c][e]);
            float m = fmaxf(0.0f, fabsf(y));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
            const int col = col_of<T, W>(lane, c, e);
            if (col < D) {
              const int b = q8_scale(m);
              a.q[row * a.ldq + col] = q8_pack1(y, q8_inverse(b));
              if ((lane & 31) == 0) a.sc[row * a.ldsc + (col >> 5)] = (uint8_t)b;
            }
          }
        }
      }
    }
  }
}

template <int XT, int RT>
__global__ __launch_bounds__(256) void rmsnorm_fwd_any_kernel(NormFwd a) {
  const int lane = threadIdx.x & 63;
  for (long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); row < a.rows; row += (long long)gridDim.x * 4) {
    auto sum = [&](int c) {
      float v = load1<XT>(a.x, row * a.ldx + c);
      if constexpr (RT != T_NONE) v += load1<RT>(a.r, row * a.ldr + c);
      return v;
    };
    float ss = 0.0f;
    for (int c = lane; c < a.D; c += 64) {
      const float v = sum(c);
      ss = fmaf(v, v, ss);
    }
    ss = wave_sum(ss);
    const float rstd = inverse_root(fmaf(ss, 1.0f / (float)a.D, a.eps));
    if (lane == 0 && a.rstd) a.rstd[row] = rstd;
    for (int c0 = 0; c0 < a.D; c0 += 64) {
      const int c = c0 + lane;
      const bool on = c < a.D;
      float y = 0.0f;
      if (on) {
        const float v = sum(c);
        if constexpr (RT != T_NONE)
          if (a.s) store1<RT>(a.s, row * a.lds + c, v);
        y = v * rstd * a.w[c];
        if (a.y) store1_by(a.y_type, a.y, row * a.ldy + c, y);
      }
      if (a.q) {
        y = q8_clean(y);
        float m = fmaxf(0.0f, fabsf(y));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        if (on) {
          const int b = q8_scale(m);
          a.q[row * a.ldq + c] = q8_pack1(y, q8_inverse(b));
          if ((lane & 31) == 0) a.sc[row * a.ldsc + (c >> 5)] = (uint8_t)b;
        }
      }
    }
  }
}

struct NormBwd {
  const void *dy, *s;
  const uint8_t* sc;
  const float *rstd, *w;
  const void* dres;
  void* dx;
  float* part;  // [gridDim.x][D]
  long long lddy, lds, ldsc, lddres, lddx, rows;
  int D, dx_type;
};

template <int ST>
__device__ __forceinline__ float load_s1(const NormBwd& a, long long row, int col) {
  if constexpr (ST == T_Q8)
    return q8_unpack1(((const uint8_t*)a.s)[row * a.lds + col], q8_value(a.sc[row * a.ldsc + (col >> 5)]));
  else
    return load1<ST>(a.s, row * a.lds + col);
}
template <int ST, int T, int W>
__device__ __forceinline__ void load_s_chunk(const NormBwd& a, long long row, int lane, int c, float* v) {
  if constexpr (ST != T_Q8) {
    load_chunk<ST, T, W>(a.s, row * a.lds, lane, c, a.D, v);
  } else if constexpr (W == 8) {
    int col = col_of<T, W>(lane, c, 0);
    col = col < a.D ? col : 0;
    const u32x2 q = *(const u32x2*)((const uint8_t*)a.s + row * a.lds + col);
    const float k = q8_value(a.sc[row * a.ldsc + (col >> 5)]);
    q8_unpack4(q[0], k, v);
    q8_unpack4(q[1], k, v + 4);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int col = col_of<T, W>(lane, c, e);
      v[e] = load_s1<ST>(a, row, col < a.D ? col : 0);
    }
  }
}

template <int DT, int ST, int T, int NCH, int W>
__global__ __launch_bounds__(256) void rmsnorm_bwd_kernel(NormBwd a) {
  constexpr int RPB = 256 / T;
  __shared__ float red[4];
  __shared__ float fold[RPB > 1 ? 256 * 8 * NCH : 1];
  const int lane = threadIdx.x % T, sub = threadIdx.x / T;
  const float inv_d = 1.0f / (float)a.D;
  float w[NCH][8], dw[NCH][8];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    load_chunk<T_F32, T, W>(a.w, 0, lane, c, a.D, w[c]);
    cut_chunk<T, W>(lane, c, a.D, w[c]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[c][e] = 0.0f;
  }
  const long long last = (a.rows + RPB - 1) / RPB * RPB;
  for (long long row = (long long)blockIdx.x * RPB + sub; row < last; row += (long long)gridDim.x * RPB) {
    const int D = row < a.rows ? a.D : 0;  // (a row past the end has no columns; it loads the last row's)
    const long long from = row < a.rows ? row : a.rows - 1;
    const float rstd = a.rstd[from];
    float g[NCH][8], n[NCH][8], o[NCH][8];
    float dot = 0.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      load_chunk<DT, T, W>(a.dy, from * a.lddy, lane, c, a.D, g[c]);
      load_s_chunk<ST, T, W>(a, from, lane, c, n[c]);
    }
    if (!a.dres) {
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) o[c][e] = 0.0f;
    } else if (a.dx_type == T_BF16) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) load_chunk<T_BF16, T, W>(a.dres, from * a.lddres, lane, c, a.D, o[c]);
    } else if (a.dx_type == T_F32) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) load_chunk<T_F32, T, W>(a.dres, from * a.lddres, lane, c, a.D, o[c]);
    } else {
#pragma unroll
      for (int c = 0; c < NCH; ++c) load_chunk<T_F16, T, W>(a.dres, from * a.lddres, lane, c, a.D, o[c]);
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      cut_chunk<T, W>(lane, c, D, g[c]);
      cut_chunk<T, W>(lane, c, D, n[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        n[c][e] *= rstd;
        dw[c][e] = fmaf(g[c][e], n[c][e], dw[c][e]);
        g[c][e] *= w[c][e];
        dot = fmaf(g[c][e], n[c][e], dot);
      }
    }
    dot = group_total<T>(dot, red) * inv_d;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) o[c][e] += rstd * (g[c][e] - n[c][e] * dot);
      store_chunk_by<T, W>(a.dx_type, a.dx, row * a.lddx, lane, c, D, o[c]);
    }
  }
  if constexpr (RPB > 1) {
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) fold[(sub * NCH + c) * T * 8 + e * T + lane] = dw[c][e];
    __syncthreads();
    if (sub == 0) {
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int k = 1; k < RPB; ++k) dw[c][e] += fold[(k * NCH + c) * T * 8 + e * T + lane];
    }
  }
  if (sub == 0) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) store_chunk<T_F32, T, W>(a.part, (long long)blockIdx.x * a.D, lane, c, a.D, dw[c]);
  }
}

template <int DT, int ST>
__global__ __launch_bounds__(256) void rmsnorm_bwd_any_kernel(NormBwd a) {
  const int lane = threadIdx.x & 63;
  for (long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); row < a.rows; row += (long long)gridDim.x * 4) {
    const float rstd = a.rstd[row];
    float dot = 0.0f;
    for (int c = lane; c < a.D; c += 64)
      dot = fmaf(load1<DT>(a.dy, row * a.lddy + c) * a.w[c], load_s1<ST>(a, row, c) * rstd, dot);
    dot = wave_sum(dot) / (float)a.D;
    for (int c = lane; c < a.D; c += 64) {
      float o = rstd * (load1<DT>(a.dy, row * a.lddy + c) * a.w[c] - load_s1<ST>(a, row, c) * rstd * dot);
      if (a.dres)
        o += a.dx_type == T_BF16 ? load1<T_BF16>(a.dres, row * a.lddres + c)
             : a.dx_type == T_F32 ? load1<T_F32>(a.dres, row * a.lddres + c)
                                  : load1<T_F16>(a.dres, row * a.lddres + c);
      store1_by(a.dx_type, a.dx, row * a.lddx + c, o);
    }
  }
}
// dw for those: workgroup (x, y) adds the rows y, y + gridDim.y, .. of 64 columns, four rows at a time. Runs before
// the kernel above, which may write dx over dy
template <int DT, int ST>
__global__ __launch_bounds__(256) void rmsnorm_dw_any_kernel(NormBwd a) {
  __shared__ float fold[4][64];
  const int lane = threadIdx.x & 63, sub = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float t = 0.0f;
  if (c < a.D)
    for (long long row = (long long)blockIdx.y * 4 + sub; row < a.rows; row += (long long)gridDim.y * 4)
      t = fmaf(load1<DT>(a.dy, row * a.lddy + c), load_s1<ST>(a, row, c) * a.rstd[row], t);
  fold[sub][lane] = t;
  __syncthreads();
  if (sub == 0 && c < a.D)
    a.part[(long long)blockIdx.y * a.D + c] = fold[0][lane] + fold[1][lane] + fold[2][lane] + fold[3][lane];
}

// dw from the workgroups' partial rows (none: zero)
__global__ __launch_bounds__(256) void dw_sum_kernel(const float* part, int rows, int D, float* dw) {
  column_sums(part, rows, D, blockIdx.x * SUM_COLS, dw);
}

constexpr int MAX_BLOCKS = 512;  // workgroups of the backward, i.e. partial rows of dw

bool vec_ok(const void* p, long long ld, int bytes) { return !p || (ld % 8 == 0 && aligned(p, bytes)); }

// T, NCH, W by width: the fewest registers that hold the row (a wave's lanes are split over rows up to 256 columns;
// single elements need the 32 lanes of an 8-bit group)
#define BY_WIDTH(D, VEC, GO)                                      \
  if (VEC) {                                                      \
    if ((D) <= 128) { GO(16, 1, 8) }                              \
    else if ((D) <= 256) { GO(32, 1, 8) }                         \
    else if ((D) <= 512) { GO(64, 1, 8) }                         \
    else if ((D) <= 1024) { GO(64, 2, 8) }                        \
    else if ((D) <= 1536) { GO(64, 3, 8) }                        \
    else if ((D) <= 2048) { GO(64, 4, 8) }                        \
    else if ((D) <= 4096) { GO(256, 2, 8) }                       \
    else { GO(256, 4, 8) }                                        \
  } else {                                                        \
    if ((D) <= 256) { GO(32, 1, 1) }                              \
    else if ((D) <= 512) { GO(64, 1, 1) }                         \
    else if ((D) <= 1024) { GO(64, 2, 1) }                        \
    else if ((D) <= 2048) { GO(64, 4, 1) }                        \
    else { GO(256, 4, 1) }                                        \
  }
constexpr int MAX_D = 8192;  // widest row that is held in registers

template <int XT, int RT>
void launch_fwd(const NormFwd& a, bool vec, hipStream_t s) {
  if (a.D > MAX_D) {
    const long long nb = (a.rows + 3) / 4;
    hipLaunchKernelGGL((rmsnorm_fwd_any_kernel<XT, RT>), dim3((unsigned)(nb < 65536 ? nb : 65536)), dim3(256), 0, s, a);
    return;
  }
#define GO(T, NCH, W)                                                                                            \
  const long long nb = (a.rows + 256 / T - 1) / (256 / T);                                                       \
  hipLaunchKernelGGL((rmsnorm_fwd_kernel<XT, RT, T, NCH, W>), dim3((unsigned)(nb < 65536 ? nb : 65536)), dim3(256), 0, s, a);
  BY_WIDTH(a.D, vec, GO)
#undef GO
}

template <int DT, int ST>
void launch_bwd(const NormBwd& a, bool vec, int nb, hipStream_t s) {
  if (a.D > MAX_D) {
    hipLaunchKernelGGL((rmsnorm_dw_any_kernel<DT, ST>), dim3((unsigned)((a.D + 63) / 64), (unsigned)nb), dim3(256), 0, s, a);
    const long long n = (a.rows + 3) / 4;
    hipLaunchKernelGGL((rmsnorm_bwd_any_kernel<DT, ST>), dim3((unsigned)(n < 65536 ? n : 65536)), dim3(256), 0, s, a);
    return;
  }
#define GO(T, NCH, W) hipLaunchKernelGGL((rmsnorm_bwd_kernel<DT, ST, T, NCH, W>), dim3((unsigned)nb), dim3(256), 0, s, a);
  BY_WIDTH(a.D, vec, GO)
#undef GO
}

// widest rows: the forward's columns count up in steps of 64 to below 2^31; a launch has fewer than 2^32 threads in a
// dimension, 256 for 64 columns of rmsnorm_dw_any_kernel and for SUM_COLS of dw_sum_kernel (where there is more than one
// partial row, or none)
constexpr int MAX_FWD_D = 0x7fffffff - 63, MAX_BWD_D = (1 << 30) - 64, MAX_SUM_D = (1 << 28) - SUM_COLS;

int bwd_blocks(int64_t rows) {
  const int64_t n = (rows + 15) / 16;
  return (int)(n < 1 ? 1 : n < MAX_BLOCKS ? n : MAX_BLOCKS);
}

}  // namespace

extern "C" int octsam_rmsnorm_fwd(const void* x, int32_t x_type, int64_t ldx, const void* r, int32_t r_type, int64_t ldr,
                                  const float* w, int64_t rows, int32_t D, float eps, void* sum_out, int64_t ld_sum, void* y,
                                  int32_t y_type, int64_t ldy, void* q, int64_t ldq, void* scale, int64_t ld_scale,
                                  float* rstd, void* stream) {
  OCTSAM_CHECK_ARG(type_ok(x_type) && (!r || type_ok(r_type)) && (!y || type_ok(y_type)), "rmsnorm_fwd: unknown type");
  OCTSAM_CHECK_ARG(rows >= 0 && D > 0 && rows <= (1ll << 40), "rmsnorm_fwd: rows %lld, D %d", (long long)rows, D);
  OCTSAM_CHECK_ARG(D <= MAX_FWD_D, "rmsnorm_fwd: D at most %d, got %d", MAX_FWD_D, D);
  if (rows == 0) return 0;
  OCTSAM_CHECK_ARG(x && w, "rmsnorm_fwd: null operand");
  OCTSAM_CHECK_ARG(!r || r_type == x_type || r_type == T_F32, "rmsnorm_fwd: the residual is fp32 or of x's type");
  OCTSAM_CHECK_ARG(!sum_out || r, "rmsnorm_fwd: sum_out without a residual");
  OCTSAM_CHECK_ARG(!q == !scale, "rmsnorm_fwd: q and scale go together");
  OCTSAM_CHECK_ARG(y || q || sum_out || rstd, "rmsnorm_fwd: no output");
  OCTSAM_CHECK_ARG(ldx >= D && (!r || ldr >= D) && (!sum_out || ld_sum >= D) && (!y || ldy >= D) &&
                       (!q || (ldq >= D && ld_scale >= (D + 31) / 32)),
                   "rmsnorm_fwd: a row stride is below the row's width");
  OCTSAM_CHECK_ARG(aligned(x, type_size(x_type)) && (!r || (aligned(r, type_size(r_type)) && aligned(sum_out, type_size(r_type)))) &&
                       (!y || aligned(y, type_size(y_type))) && aligned(w, 4) && aligned(rstd, 4),
                   "rmsnorm_fwd: an operand is not aligned to its type");
  const NormFwd a = {x, r, w, sum_out, y, (uint8_t*)q, (uint8_t*)scale, rstd, ldx, ldr, ld_sum, ldy, ldq, ld_scale, rows, D,
                     y_type, eps};
  const bool vec = D % 8 == 0 && vec_ok(x, ldx, 16) && vec_ok(r, ldr, 16) && vec_ok(sum_out, ld_sum, 16) &&
                   vec_ok(y, ldy, 16) && vec_ok(q, ldq, 8) && aligned(w, 16);
  const hipStream_t s = (hipStream_t)stream;
#define RUN(XT)                                              \
  if (!r) launch_fwd<XT, T_NONE>(a, vec, s);                 \
  else if (r_type == XT) launch_fwd<XT, XT>(a, vec, s);      \
  else launch_fwd<XT, T_F32>(a, vec, s);
  if (x_type == T_BF16) { RUN(T_BF16) } else if (x_type == T_F32) { RUN(T_F32) } else { RUN(T_F16) }
#undef RUN
  OCTSAM_LAUNCH_CHECK("octsam_rmsnorm_fwd");
  return 0;
}

extern "C" int64_t octsam_rmsnorm_bwd_workspace(int64_t rows, int32_t D) {
  if (rows < 0 || D <= 0) return 0;
  const int nb = bwd_blocks(rows);
  return nb == 1 ? 0 : (int64_t)nb * D * (int64_t)sizeof(float);
}

extern "C" int octsam_rmsnorm_bwd(const void* dy, int32_t dy_type, int64_t lddy, const void* s, int32_t s_type, int64_t lds,
                                  const void* s_scale, int64_t ld_scale, const float* rstd, const float* w, int64_t rows,
                                  int32_t D, const void* dres, int64_t lddres, void* dx, int32_t dx_type, int64_t lddx,
                                  float* dw, void* workspace, int64_t workspace_bytes, void* stream) {
  OCTSAM_CHECK_ARG(type_ok(dy_type) && type_ok(dx_type) && (type_ok(s_type) || s_type == T_Q8), "rmsnorm_bwd: unknown type");
  OCTSAM_CHECK_ARG(rows >= 0 && D > 0 && rows <= (1ll << 40), "rmsnorm_bwd: rows %lld, D %d", (long long)rows, D);
  const int most = rows == 0 || bwd_blocks(rows) > 1 ? MAX_SUM_D : MAX_BWD_D;
  OCTSAM_CHECK_ARG(D <= most, "rmsnorm_bwd: D at most %d for %lld rows, got %d", most, (long long)rows, D);
  OCTSAM_CHECK_ARG(dw, "rmsnorm_bwd: null operand");
  const hipStream_t st = (hipStream_t)stream;
  if (rows == 0) {
    hipLaunchKernelGGL(dw_sum_kernel, dim3((unsigned)((D + SUM_COLS - 1) / SUM_COLS)), dim3(256), 0, st, (const float*)nullptr, 0, D, dw);
    OCTSAM_LAUNCH_CHECK("octsam_rmsnorm_bwd");
    return 0;
  }
  OCTSAM_CHECK_ARG(dy && s && rstd && w && dx, "rmsnorm_bwd: null operand");
  OCTSAM_CHECK_ARG((s_type == T_Q8) == (s_scale != nullptr), "rmsnorm_bwd: scales come with an 8-bit s, and only with it");
  OCTSAM_CHECK_ARG(lddy >= D && lds >= D && lddx >= D && (!dres || lddres >= D) && (!s_scale || ld_scale >= (D + 31) / 32),
                   "rmsnorm_bwd: a row stride is below the row's width");
  OCTSAM_CHECK_ARG(aligned(dy, type_size(dy_type)) && (s_type == T_Q8 || aligned(s, type_size(s_type))) &&
                       aligned(dx, type_size(dx_type)) && aligned(dres, type_size(dx_type)) && aligned(w, 4) &&
                       aligned(rstd, 4) && aligned(dw, 4),
                   "rmsnorm_bwd: an operand is not aligned to its type");
  const int nb = bwd_blocks(rows);
  OCTSAM_CHECK_ARG(nb == 1 || (workspace && aligned(workspace, 16) && workspace_bytes >= octsam_rmsnorm_bwd_workspace(rows, D)),
                   "rmsnorm_bwd: the workspace needs %lld bytes, 16-B aligned", (long long)octsam_rmsnorm_bwd_workspace(rows, D));
  const NormBwd a = {dy, s, (const uint8_t*)s_scale, rstd, w, dres, dx, nb == 1 ? dw : (float*)workspace,
                     lddy, lds, ld_scale, lddres, lddx, rows, D, dx_type};
  const bool vec = D % 8 == 0 && vec_ok(dy, lddy, 16) && vec_ok(s, lds, s_type == T_Q8 ? 8 : 16) &&
                   vec_ok(dres, lddres, 16) && vec_ok(dx, lddx, 16) && aligned(w, 16) && aligned(a.part, 16);
#define RUN(DT)                                                 \
  if (s_type == T_BF16) launch_bwd<DT, T_BF16>(a, vec, nb, st); \
  else if (s_type == T_F32) launch_bwd<DT, T_F32>(a, vec, nb, st); \
  else if (s_type == T_F16) launch_bwd<DT, T_F16>(a, vec, nb, st); \
  else launch_bwd<DT, T_Q8>(a, vec, nb, st);
  if (dy_type == T_BF16) { RUN(T_BF16) } else if (dy_type == T_F32) { RUN(T_F32) } else { RUN(T_F16) }
#undef RUN
  if (nb > 1)
    hipLaunchKernelGGL(dw_sum_kernel, dim3((unsigned)((D + SUM_COLS - 1) / SUM_COLS)), dim3(256), 0, st, (const float*)workspace, nb, D, dw);
  OCTSAM_LAUNCH_CHECK("octsam_rmsnorm_bwd");
  return 0;
}
