// Gated feed-forward unit: both projections, the activation and the product in one kernel, and its backward pass.
//
//   [g | u] = x W^T + b   (W [2F, D]: F gate rows, then F up rows);   h = act(g) * u
//   dg = dh * u * act'(g);  du = dh * act(g);  dx = [dg | du] W;  dW = [dg | du]^T x;  db = column sums of [dg | du]
//
// Operands are bf16 or fp16, products accumulate in fp32 on the matrix cores, g and u stay fp32 until h (and, on
// request, g and u themselves, in 16 bits or in the 8-bit form of q8.h) is rounded once. The backward reads g and u as
// they were kept and rounds [dg | du] to the operand type before the two products (their operands are 16-bit: half a
// step, 2^-9 relative in bf16, against results that are rounded to the same step); db is summed from the unrounded
// fp32 values.
//
// All tiles run 16x16x32 MFMAs with swapped operands (a lane holds 4 consecutive columns of a row; one permlane16_swap
// makes 8). In the forward a wave's 64 columns are 32 gate rows and the 32 up rows of the same features, so a lane has g
// and u of the same 8 features and four lanes hold an 8-bit group. Operands with k contiguous and operands stored
// [k][x] (W in dx, both in dW) use the same loops: the second kind is read from LDS with the transposing 64-bit read.
#include "q8.h"
#include <math.h>
#include <type_traits>
#include "../../include/octsam.h"

namespace {
using namespace octsam;
constexpr int T_NONE = -1, T_Q8 = 3;
constexpr int OCT_SILU = OCTSAM_ACT_SILU, OCT_GELU = OCTSAM_ACT_GELU, OCT_RELU = OCTSAM_ACT_RELU;

enum Mode { GATED, NN, TN };  // A [M][K] B [N][K] gated;  A [M][K] B [K][N];  A [K][M] B [K][N]

struct GatedP {
  const void *A, *B;
  const float* bias;
  void *C, *save;
  uint8_t* scale;
  long long lda, ldb, ldc, ldsave, ldscale;
  long long split_stride;  // elements between the fp32 partials of two K splits
  int M, N, K;             // GATED: N = F
  int act, save_type, c_type, kper;
};

template <int TY>
__device__ __forceinline__ f32x4 mma(typename Elem<TY>::v8 a, typename Elem<TY>::v8 b, f32x4 c) {
  if constexpr (TY == T_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// act(g) and, with GRAD, act'(g). The reciprocal is the hardware's (1 fp32 step). GELU's distribution function is 1 - q or q
// with q = P(-|g|) = exp(-g^2 / 2) t (C1 + .. + C8 t^7), t = 1 / (1 + TP |g|): the coefficients are this library's own
// relative minimax fit of exp(x^2) erfc(x) / 2, x = |g| / sqrt 2, over |g| <= 14.5 (9.8e-8, by reweighted least squares),
// so that the left tail keeps its relative precision until the exponential leaves the normal numbers at -13.2: 36 + 1.5 g^2
// half steps of fp32 at most, most of them the exponent's. (A form with an absolute bound, as gelu_fast uses, is 0.05 % off at
// -4 and 1 % at -8, more than half a step of fp16 and bf16.)
namespace tail_c {
constexpr float TP = 0.305f, C1 = 0.12164024f, C2 = 0.1224587f, C3 = 0.10347359f, C4 = 0.120840795f, C5 = -0.037621543f,
                C6 = 0.18531598f, C7 = -0.15274678f, C8 = 0.03663905f, E = -0.5f * 1.4426950408889634f;
}
template <bool GRAD>
__device__ __forceinline__ float act_value(int act, float g, float& slope) {
  if (act == OCT_SILU) {
    const float p = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f));
    if constexpr (GRAD) slope = p * fmaf(g, 1.0f - p, 1.0f);
    return g * p;
  }
  if (act == OCT_GELU) {
    using namespace tail_c;
    const float t = __builtin_amdgcn_rcpf(fmaf(TP, fabsf(g), 1.0f));
    float c = fmaf(t, C8, C7);
    c = fmaf(c, t, C6);
    c = fmaf(c, t, C5);
    c = fmaf(c, t, C4);
    c = fmaf(c, t, C3);
    c = fmaf(c, t, C2);
    c = fmaf(c, t, C1);
    const float ex = __builtin_amdgcn_exp2f(g * E * g), q = c * t * ex;
    const float cdf = g < 0.0f ? q : 1.0f - q;
    if constexpr (GRAD) slope = fmaf(g * 0.3989422804014327f, ex, cdf);
    return g * cdf;
  }
  if (act == OCT_RELU) {
    if constexpr (GRAD) slope = g > 0.0f ? 1.0f : 0.0f;
    return g < 0.0f ? 0.0f : g;
  }
  if constexpr (GRAD) slope = 1.0f;
  return g;
}

// a lane's 8 consecutive columns of its row from two 16x16 blocks of the swapped product: columns
// 16 (q & 1) + 8 (q >> 1) .. + 7 of the 32, q = lane >> 4
__device__ __forceinline__ void row8(f32x4 a, f32x4 b, float* v) {
  const u32x4 x = __builtin_bit_cast(u32x4, a), y = __builtin_bit_cast(u32x4, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t xi = x[i], yi = y[i];
    const auto r = __builtin_amdgcn_permlane16_swap(xi, yi, false, false);
    v[i] = __builtin_bit_cast(float, (uint32_t)r[0]);
    v[4 + i] = __builtin_bit_cast(float, (uint32_t)r[1]);
  }
}

// the largest of v over the four lanes (16 apart) that hold an 8-bit group: both results of a swap of v with itself hold
// one half's values in both halves
__device__ __forceinline__ float group_max(float v) {
  const uint32_t a = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const uint32_t b = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])));
  const auto t = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)t[0]), __builtin_bit_cast(float, (uint32_t)t[1]));
}
__device__ __forceinline__ void keep8_q(const GatedP& p, long long m, int half, int f, bool ok, const float* v) {
  float a = 0.0f, w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    w[e] = q8_clean(v[e]);
    a = fmaxf(a, fabsf(w[e]));
  }
  a = group_max(ok ? a : 0.0f);
  if (ok) {
    const int b = q8_scale(a);
    const float inv = q8_inverse(b);
    *(u32x2*)((uint8_t*)p.save + m * p.ldsave + (long long)half * p.N + f) = (u32x2){q8_pack4(w, inv), q8_pack4(w + 4, inv)};
    if ((f & 31) == 0) p.scale[m * p.ldscale + half * ((p.N + 31) / 32) + (f >> 5)] = (uint8_t)b;
  }
}

struct Bias8 {
  float g[8], u[8];
};
__device__ __forceinline__ Bias8 load_bias(const GatedP& p, int f) {
  Bias8 b = {};
  if (p.bias && f < p.N) {
    load8<T_F32>(p.bias, f, b.g);
    load8<T_F32>(p.bias, (long long)p.N + f, b.u);
  }
  return b;
}

// g, u: a lane's 8 features from f on of row m (all lanes of a wave call this together). Rows past M and features
// past F (a multiple of 8) are dropped; f % 32 is the same in the four lanes that hold an 8-bit group
template <int TY>
__device__ __forceinline__ void gated_store(const GatedP& p, long long m, int f, const Bias8& b, float* g, float* u) {
  const bool ok = m < p.M && f < p.N;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    g[e] += b.g[e];
    u[e] += b.u[e];
  }
  if (p.save_type == T_Q8) {
    keep8_q(p, m, 0, f, ok, g);
    keep8_q(p, m, 1, f, ok, u);
  } else if (p.save_type != T_NONE && ok) {
    store8<TY>(p.save, m * p.ldsave + f, g);
    store8<TY>(p.save, m * p.ldsave + p.N + f, u);
  }
  float h[8], unused;
  if (p.act == OCT_SILU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = act_value<false>(OCT_SILU, g[e], unused) * u[e];
  } else if (p.act == OCT_GELU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = act_value<false>(OCT_GELU, g[e], unused) * u[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = act_value<false>(p.act, g[e], unused) * u[e];
  }
  if (ok) store8<TY>(p.C, m * p.ldc + f, h);
}

template <int TY>
__device__ __forceinline__ void plain_store(const GatedP& p, long long m, int n, int split, const float* v) {
  if (m >= p.M || n >= p.N) return;
  const long long at = m * p.ldc + n;
  if (p.c_type == T_F32) store8<T_F32>((float*)p.C + split * p.split_stride, at, v);
  else store8<TY>(p.C, at, v);
}

// ------------------------------------------------------------------------------------- 64 x 64 and 128 x 128 tiles
// LDS images. Rows of k (KC): [T rows][128 B], 16-B chunk c of row r at c ^ (r >> 1) & 7: the 16 rows of a fragment read
// land on 16 slots. [k][x] (KM): [64 rows][2 T B]; a transposing read takes four rows q and two groups of rows (r bit 3)
// at once: T = 64, two rows to 256 bytes, the swizzle gives them 4 slot pairs; T = 128, 8 slot pairs.
__device__ __forceinline__ int kc_at(int r, int c) { return r * 128 + ((c ^ ((r >> 1) & 7)) << 4); }
template <int T>
__device__ __forceinline__ int km_at(int r, int c) {
  if constexpr (T == 64) return r * 128 + ((c ^ ((r & 2) | ((r >> 1) & 4))) << 4);
  else return r * 256 + ((c ^ (((r & 3) << 2) | ((r >> 2) & 2))) << 4);
}

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// the 16 x 32 fragment of rows (columns of a KM image) x0 .. x0 + 15, k half kh
template <int TY, bool KM, int T>
__device__ __forceinline__ typename Elem<TY>::v8 fragment(const char* img, int x0, int kh, int lane) {
  typedef typename Elem<TY>::v8 v8;
  if constexpr (!KM) {
    return *(const v8*)(img + kc_at(x0 + (lane & 15), kh * 4 + (lane >> 4)));
  } else {
    const int g = lane >> 4, i = lane & 15, q = i >> 2, pp = i & 3;
    const char* at = img + km_at<T>(kh * 32 + 8 * g + q, (x0 >> 3) + (pp >> 1)) + 8 * (pp & 1);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 4 * 2 * T));  // (+4 leaves the swizzle)
    const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(v8, v);
  }
}

// T x T tiles by four waves: T = 64, 16 rows x 64 columns each; T = 128, 64 x 64 each (half the LDS reads an MFMA, where
// there are tiles enough). In the forward the columns are gate and up rows in turns of 32, T / 2 features.
template <int T>
struct TileLds {
  char stage[2][2][T * 128];  // [stage][operand]
};

// tile `tile` (column tiles first) of K split `split`
template <int TY, int MODE, int T>
__device__ __forceinline__ void tile(const GatedP& p, int tiles_n, int tile, int split, TileLds<T>& smem) {
  typedef typename Elem<TY>::v8 v8;
  constexpr bool AKM = MODE == TN, BKM = MODE != GATED;
  constexpr int AHEAD = T == 64 ? 3 : 2, NP = T / 32, MB = T == 64 ? 1 : 4, XC = T / 8;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tm = tile / tiles_n, tn = tile - tm * tiles_n;
  const long long row0 = (long long)tm * T;
  const int col0 = tn * (MODE == GATED ? T / 2 : T);
  const long long k0 = (long long)split * p.kper;
  const int kn = (int)(p.K - k0 < p.kper ? p.K - k0 : p.kper);  // (< 1: no steps, the tile is zero)
  const int steps = kn > 0 ? (kn + 63) / 64 : 0;

  // this thread's NP 16-B pieces of each operand's stage: image row r (k for KM), chunk c; at: its place in the image
  const char *pa[NP], *pb[NP];
  int ka[NP], kb[NP], la[NP], lb[NP];  // k of the piece (past K: never, where its row is none of the operand's)
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int id = tid + 256 * i;
    if constexpr (AKM) {
      const int r = id / XC, c = id % XC;
      ka[i] = row0 + c * 8 < p.M ? r : 1 << 30;
      la[i] = km_at<T>(r, c);
      pa[i] = (const char*)p.A + ((k0 + r) * p.lda + row0 + c * 8) * 2;
    } else {
      const int r = id >> 3, c = id & 7;
      ka[i] = row0 + r < p.M ? c * 8 : 1 << 30;
      la[i] = kc_at(r, c);
      pa[i] = (const char*)p.A + ((row0 + r) * p.lda + k0 + c * 8) * 2;
    }
    if constexpr (BKM) {
      const int r = id / XC, c = id % XC;
      kb[i] = col0 + c * 8 < p.N ? r : 1 << 30;
      lb[i] = km_at<T>(r, c);
      pb[i] = (const char*)p.B + ((k0 + r) * p.ldb + col0 + c * 8) * 2;
    } else {
      const int r = id >> 3, c = id & 7, f = col0 + (r >> 6) * 32 + (r & 31);  // row r: gate (r bit 5 = 0) or up row of f
      kb[i] = f < p.N ? c * 8 : 1 << 30;
      lb[i] = kc_at(r, c);
      pb[i] = (const char*)p.B + (((long long)((r >> 5) & 1) * p.N + f) * p.ldb + k0 + c * 8) * 2;
    }
  }
  const long long sa = AKM ? p.lda * 128 : 128, sb = BKM ? p.ldb * 128 : 128;
  u32x4 ra[AHEAD][NP], rb[AHEAD][NP];
  auto fetch = [&](int t, u32x4 (&a)[NP], u32x4 (&b)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      a[i] = t * 64 + ka[i] < kn ? *(const u32x4*)(pa[i] + t * sa) : (u32x4)0u;
      b[i] = t * 64 + kb[i] < kn ? *(const u32x4*)(pb[i] + t * sb) : (u32x4)0u;
    }
  };
#pragma unroll
  for (int j = 0; j < AHEAD; ++j)
    if (j < steps) fetch(j, ra[j], rb[j]);
  f32x4 acc[MB][4];
#pragma unroll
  for (int mi = 0; mi < MB; ++mi)
#pragma unroll
    for (int ni = 0; ni < 4; ++ni) acc[mi][ni] = (f32x4)0.0f;
  const int wrow = T == 64 ? wave * 16 : (wave >> 1) * 64, wcol = T == 64 ? 0 : (wave & 1) * 64;
  for (int t0 = 0; t0 < steps; t0 += AHEAD) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int t = t0 + j;
      if (t < steps) {
        char *ia = smem.stage[t & 1][0], *ib = smem.stage[t & 1][1];
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          *(u32x4*)(ia + la[i]) = ra[j][i];
          *(u32x4*)(ib + lb[i]) = rb[j][i];
        }
        if (t + AHEAD < steps) fetch(t + AHEAD, ra[j], rb[j]);
        // one barrier a step: whoever writes this buffer again has passed the next step's barrier, and so have all
        // its readers of this step
        __syncthreads();
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) {
          v8 af[MB];
#pragma unroll
          for (int mi = 0; mi < MB; ++mi) af[mi] = fragment<TY, AKM, T>(ia, wrow + mi * 16, kh, lane);
#pragma unroll
          for (int ni = 0; ni < 4; ++ni) {
            const v8 bf = fragment<TY, BKM, T>(ib, wcol + ni * 16, kh, lane);
#pragma unroll
            for (int mi = 0; mi < MB; ++mi) acc[mi][ni] = mma<TY>(bf, af[mi], acc[mi][ni]);
          }
        }
      }
    }
  }
  const int q = lane >> 4, cofs = 16 * (q & 1) + 8 * (q >> 1);
  Bias8 b;
  if constexpr (MODE == GATED) b = load_bias(p, col0 + wcol / 2 + cofs);
#pragma unroll
  for (int mi = 0; mi < MB; ++mi) {
    const long long m = row0 + wrow + mi * 16 + (lane & 15);
    float v0[8], v1[8];
    row8(acc[mi][0], acc[mi][1], v0);
    row8(acc[mi][2], acc[mi][3], v1);
    if constexpr (MODE == GATED) {
      gated_store<TY>(p, m, col0 + wcol / 2 + cofs, b, v0, v1);
    } else {
      plain_store<TY>(p, m, col0 + wcol + cofs, split, v0);
      plain_store<TY>(p, m, col0 + wcol + 32 + cofs, split, v1);
    }
  }
}

template <int TY, int T>
__global__ __launch_bounds__(256) void gated_tile_kernel(GatedP p, int tiles_n) {
  __shared__ __attribute__((aligned(16))) TileLds<T> smem;
  tile<TY, GATED, T>(p, tiles_n, blockIdx.x, 0, smem);
}

// work items go to the XCDs (workgroup id mod 8) in contiguous runs
__device__ __forceinline__ int tile_of(int bid, int nwg) {
  const int q = nwg >> 3, r = nwg & 7, xcd = bid & 7, loc = bid >> 3;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + loc;
}

// Both products of the backward in one launch, the one with the longer K runs first: its tiles (each K split of all tiles
// in turn), then the other's, which fill the gaps at the end (8192 x 768 x 2048 uncut: 154 us against 218). A run's
// tiles share their rows' panel and most of a split's columns in an XCD's L2: 2 to 6 % against tiles in the
// workgroups' order (2048 x 1024 x 2736 102 -> 96 us). (The forward's tiles, with few rows, are as fast without.)
struct TileJob {
  GatedP p;
  int tiles, tiles_n, splits;
};
template <int TY, int T>
__global__ __launch_bounds__(256) void gated_pair_kernel(TileJob x, TileJob w, bool w_first) {
  __shared__ __attribute__((aligned(16))) TileLds<T> smem;
  const int nx = x.tiles * x.splits, nw = w.tiles * w.splits, from = w_first ? nw : 0;  // where dx's workgroups start
  int b = blockIdx.x;
  if (b >= from && b < from + nx) {
    b = tile_of(b - from, nx);
    tile<TY, NN, T>(x.p, x.tiles_n, b % x.tiles, b / x.tiles, smem);
  } else {
    b = tile_of(w_first ? b : b - nx, nw);
    tile<TY, TN, T>(w.p, w.tiles_n, b % w.tiles, b / w.tiles, smem);
  }
}

// ----------------------------------------------------------------------------------------------- for the large tiles
constexpr int OUT_OF_RANGE = (int)0x80000000;

__device__ __forceinline__ void hard_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t range(const void* base, long long bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)(bytes > 0 ? bytes : 0), 0x00020000);
}

// within a run eight row tiles take turns over the column tiles, so that what is in flight on an XCD shares row and column
// panels in its L2
__device__ __forceinline__ void place(int id, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int per = 8 * tiles_n, g = id / per, in = id - g * per;
  const int h = tiles_m - g * 8 < 8 ? tiles_m - g * 8 : 8;
  tn = in / h;
  tm = g * 8 + (in - tn * h);
}

// ------------------------------------------------------------------------ the forward: two workgroups to a CU
// 128 rows x 128 features (256 columns) x 64 tiles, four waves of 128 x 64. LDS holds one stage of A (16 KiB) and two of B
// (64): 80 KiB, so two workgroups share a CU and each SIMD has a wave of either. A K-step is: wait for the stage; all 24
// fragments into registers; barrier; A's next stage and B's next but one on their way; 64 MFMAs. K is short here (D) and
// the epilogue long (activation, product, 8-bit groups: about 25 vector operations per element of h): while one workgroup
// is in its epilogue, its first loads, a wait or its fragment reads, the other has the matrix cores.
// 16384 x 1024 x 2736 bf16, medians with the chip kept busy: 186 us without a save (990 TFLOP/s), 206 with 16 bits, 221 with
// 8 bits (the library's plain product of this shape, a pass of each in turn: 249). Timed in turn, the 256 x 256 tiles below,
// one workgroup to a CU, took 8 % longer without a save and 7 % with 8 bits (for the backward's longer K they are ahead: dx
// took a fifth less, with two thirds of the reads).
// The fragment reads are assembly with their wait in the same block: as ordinary loads they would wait for all DMA in
// flight.
constexpr int DUO_B = 16384, DUO_LDS = 81920;

// fragments of 16-row blocks 2048 bytes apart, k half by k half (a0, a1), from rows of k
template <typename V>
__device__ __forceinline__ void read_rows(V (&f)[8][2], uint32_t a0, uint32_t a1) {
  asm volatile(
      "ds_read_b128 %0, %16\n\tds_read_b128 %1, %17\n\tds_read_b128 %2, %16 offset:2048\n\tds_read_b128 %3, %17 offset:2048\n\t"
      "ds_read_b128 %4, %16 offset:4096\n\tds_read_b128 %5, %17 offset:4096\n\t"
      "ds_read_b128 %6, %16 offset:6144\n\tds_read_b128 %7, %17 offset:6144\n\t"
      "ds_read_b128 %8, %16 offset:8192\n\tds_read_b128 %9, %17 offset:8192\n\t"
      "ds_read_b128 %10, %16 offset:10240\n\tds_read_b128 %11, %17 offset:10240\n\t"
      "ds_read_b128 %12, %16 offset:12288\n\tds_read_b128 %13, %17 offset:12288\n\t"
      "ds_read_b128 %14, %16 offset:14336\n\tds_read_b128 %15, %17 offset:14336\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(f[0][0]), "=&v"(f[0][1]), "=&v"(f[1][0]), "=&v"(f[1][1]), "=&v"(f[2][0]), "=&v"(f[2][1]), "=&v"(f[3][0]),
        "=&v"(f[3][1]), "=&v"(f[4][0]), "=&v"(f[4][1]), "=&v"(f[5][0]), "=&v"(f[5][1]), "=&v"(f[6][0]), "=&v"(f[6][1]),
        "=&v"(f[7][0]), "=&v"(f[7][1])
      : "v"(a0), "v"(a1)
      : "memory");
}
template <typename V>
__device__ __forceinline__ void read_rows(V (&f)[4][2], uint32_t a0, uint32_t a1) {
  asm volatile(
      "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %8 offset:2048\n\tds_read_b128 %3, %9 offset:2048\n\t"
      "ds_read_b128 %4, %8 offset:4096\n\tds_read_b128 %5, %9 offset:4096\n\t"
      "ds_read_b128 %6, %8 offset:6144\n\tds_read_b128 %7, %9 offset:6144\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(f[0][0]), "=&v"(f[0][1]), "=&v"(f[1][0]), "=&v"(f[1][1]), "=&v"(f[2][0]), "=&v"(f[2][1]), "=&v"(f[3][0]),
        "=&v"(f[3][1])
      : "v"(a0), "v"(a1)
      : "memory");
}
template <int TY>
__device__ __forceinline__ void duo_tile(const GatedP& p, int tiles_m, int tiles_n, char* lds) {
  typedef typename Elem<TY>::v8 v8;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  place(tile_of(blockIdx.x, gridDim.x), tiles_m, tiles_n, tm, tn);
  const long long row0 = (long long)tm * 128;
  const int col0 = tn * 128, n = (p.K + 63) / 64;
  const long long lda2 = p.lda * 2, ldb2 = p.ldb * 2;
  // a lane's part of a 1 KiB DMA piece (8 rows of 128 B), by the piece's parity: its chunk's k and its offset
  int kc[2], va[2], vb[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = e * 8 + (lane >> 3);
    kc[e] = ((lane & 7) ^ ((r >> 1) & 7)) * 8;
    va[e] = (int)(r * lda2) + kc[e] * 2;
    vb[e] = (int)(r * ldb2) + kc[e] * 2;
  }
  const int nf = p.N - col0 < 128 ? p.N - col0 : 128;
  const __amdgpu_buffer_rsrc_t ra = range((const char*)p.A + row0 * lda2, (p.M - row0 < 128 ? p.M - row0 : 128) * lda2);
  const __amdgpu_buffer_rsrc_t rg = range((const char*)p.B + (long long)col0 * ldb2, nf * ldb2);
  const __amdgpu_buffer_rsrc_t ru = range((const char*)p.B + ((long long)p.N + col0) * ldb2, nf * ldb2);
  // (only the last K-step of a K that is no multiple of 64 has chunks past K)
  auto cut = [&](int v, int e, int t) { return t * 64 + 64 <= p.K || t * 64 + kc[e] < p.K ? v : OUT_OF_RANGE; };
  auto load_a = [&](int t) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr_t)(lds + (wave * 4 + i) * 1024), 16, cut(va[i & 1], i & 1, t),
                                               (int)((wave * 32 + (i & ~1) * 8) * lda2) + t * 128, 0, 0);
  };
  auto load_b = [&](int t) {  // image rows 64 wave + (0-31: gate features 32 wave .., 32-63: the same features' up rows)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(i < 4 ? rg : ru, (lds_ptr_t)(lds + DUO_B + (t & 1) * 32768 + (wave * 8 + i) * 1024), 16,
                                               cut(vb[i & 1], i & 1, t), (int)((wave * 32 + (i & 2) * 8) * ldb2) + t * 128, 0, 0);
  };
  f32x4 acc[8][4];
#pragma unroll
  for (int mi = 0; mi < 8; ++mi)
#pragma unroll
    for (int ni = 0; ni < 4; ++ni) acc[mi][ni] = (f32x4)0.0f;
  const int fr = lane & 15;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds, row_at = fr * 128 + (((lane >> 4) ^ ((fr >> 1) & 7)) << 4);
  load_b(0);
  load_a(0);
  if (n > 1) load_b(1);
  for (int t = 0; t < n; ++t) {
    if (t + 1 < n) wait_loads<8>();  // (loads land in order: all but B(t + 1))
    else wait_loads<0>();
    hard_barrier();
    v8 af[8][2], bf[4][2];
    const uint32_t ib = lds0 + DUO_B + (t & 1) * 32768 + wave * 8192 + row_at;
    read_rows(bf, ib, ib ^ 64);
    read_rows(af, lds0 + row_at, lds0 + (row_at ^ 64));
    hard_barrier();  // (every wave has its fragments: A's stage and this one of B may be written)
    if (t + 1 < n) load_a(t + 1);
    if (t + 2 < n) load_b(t + 2);
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int mi = 0; mi < 8; ++mi)
#pragma unroll
        for (int ni = 0; ni < 4; ++ni) acc[mi][ni] = mma<TY>(bf[ni][kh], af[mi][kh], acc[mi][ni]);
  }
  const int q = lane >> 4, f = col0 + wave * 32 + 16 * (q & 1) + 8 * (q >> 1);
  const Bias8 b = load_bias(p, f);
#pragma unroll
  for (int mi = 0; mi < 8; ++mi) {
    float g[8], u[8];
    row8(acc[mi][0], acc[mi][1], g);
    row8(acc[mi][2], acc[mi][3], u);
    gated_store<TY>(p, row0 + mi * 16 + (lane & 15), f, b, g, u);
  }
}
template <int TY>
__global__ __launch_bounds__(256, 2) void gated_duo_kernel(GatedP p, int tiles_m, int tiles_n) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  duo_tile<TY>(p, tiles_m, tiles_n, lds);
}

// ----------------------------------------------------------------------------------------------------- 256 x 256 tile
// The backward's large products: 256 x 256 x 64 tiles, eight waves as 2 (rows) x 4 (columns) with 128 x 64 each, operands
// by LDS-DMA through buffer descriptors (what lies past an operand's end reads as zero), two stages of 64 KiB. A K-step of a
// wave is two segments between barriers: L reads its 24 fragments and issues its share of the DMA, C runs its 64 MFMAs; the
// two wave rows run one segment apart, so that each SIMD has one wave in its MFMAs while its other wave loads. A's rows
// 0-127 are read by wave row 0 alone (segment 2t), 128-255 by wave row 1 (2t + 1), B by both, and a region is refilled once
// its last reader has passed a barrier:
//   wave row 0 in L(t): B(t + 1), landed at the end of its C(t)
//   wave row 1 in L(t): A-hi(t + 1), landed at the end of its C(t); A-lo(t + 2), landed at the end of its L(t + 1)
//   before the loop:    stage 0 and A-lo(1)
// LDS images: rows of k as above; [k][x] operands as two halves of 128 columns, [64][256 B], chunk c of row r at
// c ^ 2 ((r & 3) << 1 | (r >> 3) & 1): a transposing read's 32 lanes (rows q of 4, and 8 + q) cover 16 chunk slots, and
// a fragment's address is one xor of a lane constant with the column block, plus constants.
// 16384 x 5472 x 1024 (dx of 16384 x 1024 x 2736): median 160 us, 1150 TFLOP/s, MFMAs busy 55 % of the cycles at the 2.06 GHz
// that the chip holds (the library's product, a pass of each in turn: 161); dw of the same sizes 185 (263). What bounds it is
// the sum of the parts on one SIMD pair: of the loop's time then (152 us), copies of the kernel with the other parts left out
// took 97 % with the DMA alone, 44 % with the fragment reads alone, 78 % with reads and MFMAs. Three stages of B did not
// shorten it, nor did 32x32x16 MFMAs; scalar work kept out of the loop (descriptors by addition, a loop for each wave row)
// and the MFMA segments' priority took a tenth off dw of 16384 x 1280 x 3416, which now takes 249 us (the library 429).
constexpr int STAGE = 65536;

template <int TY, bool KM>
__device__ __forceinline__ typename Elem<TY>::v8 frag256(const char* img, int x0, int kb, int lane) {
  typedef typename Elem<TY>::v8 v8;
  if constexpr (!KM) {
    return *(const v8*)(img + kc_at(x0 + (lane & 15), kb * 4 + (lane >> 4)));
  } else {  // img: the 128-column half, x0 < 128
    const int g = lane >> 4, q = (lane & 15) >> 2, pp = lane & 3;
    const int base = (8 * g + q) * 256 + (((q << 1) | (g & 1)) << 5) + ((pp >> 1) << 4) + 8 * (pp & 1);
    const char* at = img + (base ^ (x0 << 1)) + kb * 8192;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 1024));
    const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(v8, v);
  }
}

// A [k][x] operand's rows from K-step to K-step: the descriptor of the 64 rows at hand (fewer at K's end: the others read as
// zero), from column x0 of xdim on. Kept by addition: the loop's scalar instructions stand in the way of its loads
struct StepRows {
  const char* at;
  long long step;  // bytes of 64 rows
  int ld2, width, left;
  __device__ __forceinline__ StepRows(const void* X, long long ld, long long x0, long long xdim, int k, int K)
      : at((const char*)X + (long long)k * ld * 2 + x0 * 2), step(ld * 128), ld2((int)ld * 2), width((int)(xdim - x0) * 2), left(K - k) {}
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows() const {
    const int bytes = ((left < 64 ? left : 64) - 1) * ld2 + width;
    return __builtin_amdgcn_make_buffer_rsrc((void*)at, (short)0, bytes > 0 ? bytes : 0, 0x00020000);
  }
  __device__ __forceinline__ void next() {
    at += step;
    left -= 64;
  }
};

// acc = the tile at (row0, col0) over the K-steps [kb, kb + n), n >= 1
template <int TY, int MODE>
__device__ __forceinline__ void tile256(const GatedP& p, long long row0, int col0, int kb, int n, f32x4 (&acc)[8][4], char* lds,
                                        int wave, int lane) {
  typedef typename Elem<TY>::v8 v8;
  constexpr bool AKM = MODE == TN;  // (B is [k][x] in both)
  const int wr = wave >> 2, wc = wave & 3;
  const int lda2 = (int)p.lda * 2, ldb2 = (int)p.ldb * 2;
  // a lane's part of a 1 KiB DMA piece j. k in rows: 8 rows of 128 B, by j & 1; [k][x]: 4 rows of 256 B, by (j >> 1) & 1
  // (the part of the chunk swizzle that the piece number gives)
  int va[2], vb[2], kc[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = e * 8 + (lane >> 3);
    kc[e] = ((lane & 7) ^ ((r >> 1) & 7)) * 8;
    const int cols = ((lane & 15) ^ (((lane >> 4) << 2) | (e << 1))) << 4;
    va[e] = AKM ? (lane >> 4) * lda2 + cols : r * lda2 + kc[e] * 2;
    vb[e] = (lane >> 4) * ldb2 + cols;
  }
  StepRows sa(p.A, p.lda, row0, p.M, kb * 64, p.K), sb(p.B, p.ldb, col0, p.N, kb * 64, p.K);
  const __amdgpu_buffer_rsrc_t ra = range((const char*)p.A + row0 * p.lda * 2, (p.M - row0 < 256 ? p.M - row0 : 256) * p.lda * 2);
  // pieces [j0, j0 + N) of half h of A (16 a half), stage t; s: A's rows of that stage
  auto load_a = [&](const StepRows& s, int h, int j0, int t, auto count) __attribute__((always_inline)) {
    char* dst = lds + (t & 1) * STAGE + h * 16384 + j0 * 1024;
    const int k = (kb + t) * 64;
    int v[2] = {va[0], va[1]};
    if (!AKM && k + 64 > p.K) {  // (a K that is no multiple of 64: chunks past it)
#pragma unroll
      for (int e = 0; e < 2; ++e) v[e] = k + kc[e] < p.K ? va[e] : OUT_OF_RANGE;
    }
    const __amdgpu_buffer_rsrc_t rs = AKM ? s.rows() : ra;
    const int at = AKM ? j0 * 4 * lda2 + h * 256 : (h * 128 + j0 * 8) * lda2 + k * 2;
#pragma unroll
    for (int i = 0; i < decltype(count)::value; ++i)  // (j0 is even)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(dst + i * 1024), 16, v[AKM ? ((j0 + i) >> 1) & 1 : i & 1],
                                               at + (AKM ? i * 4 : (i & ~1) * 8) * lda2, 0, 0);
  };
  // pieces [j0, j0 + N) of B (32, 16 to a half of 128 columns; j0 a multiple of 4)
  auto load_b = [&](const StepRows& s, int j0, int t, auto count) __attribute__((always_inline)) {
    char* dst = lds + (t & 1) * STAGE + 32768 + j0 * 1024;
    const __amdgpu_buffer_rsrc_t rs = s.rows();
    const int at = (j0 & 15) * 4 * ldb2 + (j0 >> 4) * 256;
#pragma unroll
    for (int i = 0; i < decltype(count)::value; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(dst + i * 1024), 16, vb[(i >> 1) & 1], at + i * 4 * ldb2, 0, 0);
  };
  using std::integral_constant;
#pragma unroll
  for (int mi = 0; mi < 8; ++mi)
#pragma unroll
    for (int ni = 0; ni < 4; ++ni) acc[mi][ni] = (f32x4)0.0f;
  load_a(sa, 0, wave * 2, 0, integral_constant<int, 2>());
  load_a(sa, 1, wave * 2, 0, integral_constant<int, 2>());
  load_b(sb, wave * 4, 0, integral_constant<int, 4>());
  sa.next();
  sb.next();
  if (n > 1) {
    load_a(sa, 0, wave * 2, 1, integral_constant<int, 2>());
    wait_loads<2>();
  } else {
    wait_loads<0>();
  }
  hard_barrier();
  // (a loop for each wave row: nothing of one stands in the other's way)
  auto step = [&](int t, auto row) __attribute__((always_inline)) {
    constexpr int WR = decltype(row)::value;
    const char* cur = lds + (t & 1) * STAGE;
    v8 af[8][2], bf[4][2];
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
#pragma unroll
      for (int ni = 0; ni < 4; ++ni)
        bf[ni][kh] = frag256<TY, true>(cur + 32768 + (wc >> 1) * 16384, (wc & 1) * 64 + ni * 16, kh, lane);
#pragma unroll
      for (int mi = 0; mi < 8; ++mi) {
        if constexpr (AKM) af[mi][kh] = frag256<TY, true>(cur + WR * 16384, mi * 16, kh, lane);
        else af[mi][kh] = frag256<TY, false>(cur, WR * 128 + mi * 16, kh, lane);
      }
    }
    if constexpr (WR == 0) {
      if (t + 1 < n) load_b(sb, wc * 8, t + 1, integral_constant<int, 8>());
      sb.next();
    } else {
      if (t + 1 < n) load_a(sa, 1, wc * 4, t + 1, integral_constant<int, 4>());
      sa.next();
      if (t + 2 < n) load_a(sa, 0, wc * 4, t + 2, integral_constant<int, 4>());
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the fragments are in registers: the stage may be refilled)
    if constexpr (WR == 1) {
      if (t + 2 < n) wait_loads<8>();
      else if (t + 1 < n) wait_loads<4>();
      else wait_loads<0>();
    }
    hard_barrier();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int mi = 0; mi < 8; ++mi)
#pragma unroll
        for (int ni = 0; ni < 4; ++ni) acc[mi][ni] = mma<TY>(bf[ni][kh], af[mi][kh], acc[mi][ni]);
    __builtin_amdgcn_s_setprio(0);
    if constexpr (WR == 0) {
      wait_loads<0>();
      hard_barrier();
    } else {
      if (t + 2 < n) wait_loads<4>();
      else wait_loads<0>();
      if (t + 1 < n) hard_barrier();
    }
  };
  if (wr == 0) {
    for (int t = 0; t < n; ++t) step(t, integral_constant<int, 0>());
  } else {
    hard_barrier();
    for (int t = 0; t < n; ++t) step(t, integral_constant<int, 1>());
  }
}

template <int TY>
__device__ __forceinline__ void store256(const GatedP& p, long long row0, int col0, f32x4 (&acc)[8][4], int wave, int lane) {
  const int wr = wave >> 2, wc = wave & 3, q = lane >> 4, cofs = 16 * (q & 1) + 8 * (q >> 1);
#pragma unroll
  for (int mi = 0; mi < 8; ++mi) {
    const long long m = row0 + wr * 128 + mi * 16 + (lane & 15);
    float v0[8], v1[8];
    row8(acc[mi][0], acc[mi][1], v0);
    row8(acc[mi][2], acc[mi][3], v1);
    plain_store<TY>(p, m, col0 + wc * 64 + cofs, 0, v0);
    plain_store<TY>(p, m, col0 + wc * 64 + 32 + cofs, 0, v1);
  }
}

// ----------------------------------------------------------------------------------------------------- a few rows of x
// Up to 16 MB rows (serving: one token, a batch of them) the time is W's way from memory, so W is read once, straight
// into fragments and with many loads in flight: a workgroup has NF features (their gate and up rows; NF = 8: both in one
// block of 16), its eight waves take the K-steps of 32 in turn (neighbours share 128-byte lines), load 8 / MB steps at
// once, and their sums meet in LDS. Rows of x past M read as zero. NF: 32 where an 8-bit group has to stay together; else
// 8 while that makes at most one workgroup for each CU, and 16. Measured on the GPU (bf16, us, W in cache / a new W each
// call; NF = 8, 16, 32; an empty launch is about 2.5): one row, 768 x 2048 3.2 / 4.1, 3.8 / 4.6, 5.4 / 6.2;
// 1280 x 3416 5.2 / 6.3, 4.9 / 6.2, 7.5 / 9.2; 4 x 4096 x 11008 33 / 40, 32 / 41, 41 / 52 (4.3 TB/s of a new W).
constexpr int FEW_WAVES = 8;

// four consecutive features of a row, with no 8-bit save
template <int TY>
__device__ __forceinline__ void gated_store4(const GatedP& p, long long m, int f, f32x4 g, f32x4 u) {
  typedef typename Elem<TY>::t t;
  typedef t t4 __attribute__((ext_vector_type(4)));
  if (m >= p.M || f >= p.N) return;
  if (p.bias) {
    g += *(const f32x4*)(p.bias + f);
    u += *(const f32x4*)(p.bias + p.N + f);
  }
  if (p.save_type != T_NONE) {
    t4 kg, ku;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      kg[e] = (t)g[e];
      ku[e] = (t)u[e];
    }
    *(t4*)((t*)p.save + m * p.ldsave + f) = kg;
    *(t4*)((t*)p.save + m * p.ldsave + p.N + f) = ku;
  }
  t4 h;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float unused;
    h[e] = (t)(act_value<false>(p.act, g[e], unused) * u[e]);
  }
  *(t4*)((t*)p.C + m * p.ldc + f) = h;
}

template <int TY, int NF, int MB>
__global__ __launch_bounds__(64 * FEW_WAVES) void gated_few_kernel(GatedP p) {
  typedef typename Elem<TY>::v8 v8;
  constexpr int HALF = NF / 16, NB = NF == 8 ? 1 : 2 * HALF, FEW_STEPS = 8 / MB;
  __shared__ f32x4 sums[FEW_WAVES][NB][MB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int f0 = blockIdx.x * NF;
  const int steps = (p.K + 31) / 32;
  const char *px[MB], *pw[NB];
  bool ox[MB], ow[NB];
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    ox[i] = i * 16 + r < p.M;
    px[i] = (const char*)p.A + ((ox[i] ? i * 16 + r : 0) * p.lda + g * 8) * 2;
  }
#pragma unroll
  for (int i = 0; i < NB; ++i) {  // gate rows in blocks of 16, then the up rows of the same features
    const int f = NF == 8 ? f0 + (r & 7) : f0 + (i & (HALF - 1)) * 16 + r, up = NF == 8 ? r >> 3 : i >= HALF;
    ow[i] = f < p.N;
    pw[i] = (const char*)p.B + (((long long)up * p.N + (ow[i] ? f : 0)) * p.ldb + g * 8) * 2;
  }
  f32x4 acc[NB][MB];
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[j][i] = (f32x4)0.0f;
  for (int s0 = wave; s0 < steps; s0 += FEW_WAVES * FEW_STEPS) {
    u32x4 w[FEW_STEPS][NB], x[FEW_STEPS][MB];
#pragma unroll
    for (int k = 0; k < FEW_STEPS; ++k) {
      const long long at = (s0 + k * FEW_WAVES) * 64ll;
      const bool in = (s0 + k * FEW_WAVES) * 32 + g * 8 < p.K;
#pragma unroll
      for (int j = 0; j < NB; ++j) w[k][j] = in && ow[j] ? *(const u32x4*)(pw[j] + at) : (u32x4)0u;
#pragma unroll
      for (int i = 0; i < MB; ++i) x[k][i] = in && ox[i] ? *(const u32x4*)(px[i] + at) : (u32x4)0u;
    }
#pragma unroll
    for (int k = 0; k < FEW_STEPS; ++k)
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i)
          acc[j][i] = mma<TY>(__builtin_bit_cast(v8, w[k][j]), __builtin_bit_cast(v8, x[k][i]), acc[j][i]);
  }
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MB; ++i) sums[wave][j][i][lane] = acc[j][i];
  __syncthreads();
  if (wave >= MB) return;
  f32x4 v[NB];  // of the wave's 16 rows
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    v[j] = sums[0][j][wave][lane];
#pragma unroll
    for (int k = 1; k < FEW_WAVES; ++k) v[j] += sums[k][j][wave][lane];
  }
  const int m = wave * 16 + r;
  if constexpr (NF == 32) {
    const int cofs = 16 * (g & 1) + 8 * (g >> 1);
    float v0[8], v1[8];
    row8(v[0], v[1], v0);
    row8(v[2], v[3], v1);
    gated_store<TY>(p, m, f0 + cofs, load_bias(p, f0 + cofs), v0, v1);
  } else if constexpr (NF == 16) {
    gated_store4<TY>(p, m, f0 + 4 * g, v[0], v[1]);
  } else {
    f32x4 u;
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __shfl_xor(v[0][i], 32);
    if (g < 2) gated_store4<TY>(p, m, f0 + 4 * g, v[0], u);
  }
}
template <int TY, int MB>
void forward_few16(const GatedP& p, hipStream_t s) {
  if (p.N <= 8 * 256) hipLaunchKernelGGL((gated_few_kernel<TY, 8, MB>), dim3((unsigned)((p.N + 7) / 8)), dim3(64 * FEW_WAVES), 0, s, p);
  else hipLaunchKernelGGL((gated_few_kernel<TY, 16, MB>), dim3((unsigned)((p.N + 15) / 16)), dim3(64 * FEW_WAVES), 0, s, p);
}
template <int TY, int MB>
void forward_few(const GatedP& p, hipStream_t s) {
  if (p.save_type != T_Q8) return forward_few16<TY, MB>(p, s);
  hipLaunchKernelGGL((gated_few_kernel<TY, 32, MB>), dim3((unsigned)((p.N + 31) / 32)), dim3(64 * FEW_WAVES), 0, s, p);
}

// How a product's tiles meet the chip's 256 workgroups: `whole` tiles (a multiple of 256) are one workgroup's each. Of
// the `rest` others K is cut into `splits` parts, all tiles at the same places; of the rest * splits parts, in the order
// part-major, the first `wgs` are a workgroup's first job each, so that what runs together on an XCD walks the same K
// over neighbouring tiles and shares its panels in L2 (cut end to end into equal runs instead, every workgroup walked a
// K of its own: dw of 16384 x 1280 x 3416 took half as long again on the same loop). What is left, `over`
// tiles' last parts, is cut into `runs` each, the second jobs of the first over * runs workgroups: more runs end sooner
// but each leaves a partial tile of 256 KiB. All jobs leave fp32 partial tiles (slot w, then wgs + w), and
// gated_fix_kernel adds a tile's in order. wgs = 0: every tile is whole.
struct Share {
  int tiles_m, tiles_n, steps, whole, rest, splits, wgs, over, runs;
};
__device__ __host__ __forceinline__ int part_start(const Share& s, int j) { return (int)((long long)j * s.steps / s.splits); }

template <int TY, int MODE>
__global__ __launch_bounds__(512, 2) void gated_big_kernel(GatedP p, Share sh, float* part) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  f32x4 acc[8][4];
  int tm, tn;
  if ((int)blockIdx.x < sh.whole) {
    place(tile_of(blockIdx.x, sh.whole), sh.tiles_m, sh.tiles_n, tm, tn);
    tile256<TY, MODE>(p, (long long)tm * 256, tn * 256, 0, sh.steps, acc, lds, wave, lane);
    store256<TY>(p, (long long)tm * 256, tn * 256, acc, wave, lane);
    return;
  }
  const int w = tile_of(blockIdx.x - sh.whole, sh.wgs);
  GatedP q = p;  // a partial tile
  q.ldc = 256;
  q.c_type = T_F32;
  q.M = q.N = 256;
  const int j = w / sh.rest;
  int t = w - j * sh.rest, kb = part_start(sh, j), n = part_start(sh, j + 1) - kb;
  for (int slot = w;; slot = sh.wgs + w) {
    place(sh.whole + t, sh.tiles_m, sh.tiles_n, tm, tn);
    tile256<TY, MODE>(p, (long long)tm * 256, tn * 256, kb, n, acc, lds, wave, lane);
    q.C = part + (long long)slot * 65536;
    store256<TY>(q, 0, 0, acc, wave, lane);
    if (slot >= sh.wgs || w >= sh.over * sh.runs) break;
    const int l = w / sh.runs, i = w - l * sh.runs, k0 = part_start(sh, sh.splits - 1), len = sh.steps - k0;
    t = sh.rest - sh.over + l;
    kb = k0 + (int)((long long)i * len / sh.runs);
    n = k0 + (int)((long long)(i + 1) * len / sh.runs) - kb;
  }
}

// the tiles that were left in partials: workgroup (8 rows, tile)
template <int TY>
__global__ __launch_bounds__(256) void gated_fix_kernel(GatedP p, Share sh, const float* __restrict__ part) {
  const int t = blockIdx.y, r = blockIdx.x * 8 + (threadIdx.x >> 5), c = (threadIdx.x & 31) * 8;
  int tm, tn;
  place(sh.whole + t, sh.tiles_m, sh.tiles_n, tm, tn);
  const long long m = (long long)tm * 256 + r;
  const int n = tn * 256 + c;
  if (m >= p.M || n >= p.N) return;
  float v[8] = {};
  // `count` partials, `step` slots apart, four in flight
  auto add = [&](int slot, int step, int count) {
    const float* at = part + (long long)slot * 65536 + r * 256 + c;
    const long long by = (long long)step * 65536;
    int j = 0;
    for (; j + 4 <= count; j += 4) {
      float x[4][8];
#pragma unroll
      for (int i = 0; i < 4; ++i) load8<T_F32>(at, (j + i) * by, x[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += x[i][e];
    }
    for (; j < count; ++j) {
      float x[8];
      load8<T_F32>(at, j * by, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += x[e];
    }
  };
  const int l = t - (sh.rest - sh.over);  // >= 0: the last part was a second job
  add(t, sh.rest, l < 0 ? sh.splits : sh.splits - 1);
  if (l >= 0) add(sh.wgs + l * sh.runs, 1, sh.runs);
  if (p.c_type == T_F32) store8<T_F32>(p.C, m * p.ldc + n, v);
  else store8<TY>(p.C, m * p.ldc + n, v);
}

// What is left after the products, in one launch: the K splits' fp32 partials of dx and dw added in order and rounded
// once (a thread: 8 columns), and the row slabs' partial sums of db (a workgroup: SUM_COLS columns).
struct JoinJob {
  const float* part;
  void* out;
  long long stride, rows, ldo;
  int splits, nch, type;  // splits < 2: nothing to do
  unsigned blocks;
};
struct DbJob {
  const float* part;
  float* out;
  int slabs, n;
  unsigned blocks;
};
template <int TY>
__device__ __forceinline__ void join_block(const JoinJob& j, unsigned block) {
  const long long i = (long long)block * 256 + threadIdx.x;
  if (i >= j.rows * j.nch) return;
  const long long r = i / j.nch;
  float v[8], t[8];
  load8<T_F32>(j.part, i * 8, v);
  for (int s = 1; s < j.splits; ++s) {
    load8<T_F32>(j.part, s * j.stride + i * 8, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += t[e];
  }
  const long long at = r * j.ldo + (i - r * j.nch) * 8;
  if (j.type == T_F32) store8<T_F32>(j.out, at, v);
  else store8<TY>(j.out, at, v);
}
template <int TY>
__global__ __launch_bounds__(256) void gated_finish_kernel(JoinJob x, JoinJob w, DbJob d) {
  if (blockIdx.x < x.blocks) return join_block<TY>(x, blockIdx.x);
  if (blockIdx.x < x.blocks + w.blocks) return join_block<TY>(w, blockIdx.x - x.blocks);
  column_sums(d.part, d.slabs, d.n, (blockIdx.x - x.blocks - w.blocks) * SUM_COLS, d.out);
}

// --------------------------------------------------------------------------------------------- element-wise backward
struct ActBwd {
  const void *dh, *gu;
  const uint8_t* gs;
  void *dgu, *h;
  float* part;  // [gridDim.y][2F], or null
  long long lddh, ldgu, ldgs, lddgu, ldh, M;
  long long slab;
  int F, act;
  const void* x8;  // an 8-bit x to be read back into x16 [M][D], or null
  const uint8_t* xs;
  void* x16;
  long long ldx, ldxs;
  int D;
};

// workgroup (x, y): 256 features (32 lanes of 8) of the rows [y * slab, (y + 1) * slab), eight rows at a time; behind
// the features' workgroups, those that read 256 columns of an 8-bit x back for dw's product
template <int TY, int ST>
__global__ __launch_bounds__(256) void gated_act_bwd_kernel(ActBwd a) {
  __shared__ float fold[8][16][33];
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5, feature_blocks = (a.F + 255) / 256;
  if ((int)blockIdx.x >= feature_blocks) {
    const int c = (blockIdx.x - feature_blocks) * 256 + lane * 8;
    const long long r0 = (long long)blockIdx.y * a.slab, r1 = r0 + a.slab < a.M ? r0 + a.slab : a.M;
    for (long long r = r0 + sub; r < r1 && c < a.D; r += 8) {
      const u32x2 q = *(const u32x2*)((const uint8_t*)a.x8 + r * a.ldx + c);
      const float k = q8_value(a.xs[r * a.ldxs + (c >> 5)]);
      float v[8];
      q8_unpack4(q[0], k, v);
      q8_unpack4(q[1], k, v + 4);
      store8<TY>(a.x16, r * a.D + c, v);
    }
    return;
  }
  const int f = blockIdx.x * 256 + lane * 8;
  const bool on = f < a.F;
  float db[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) db[e] = 0.0f;
  const long long r0 = (long long)blockIdx.y * a.slab, r1 = r0 + a.slab < a.M ? r0 + a.slab : a.M;
  for (long long r = r0 + sub; r < r1 && on; r += 8) {
    float g[8], u[8], d[8], h[8];
    load8<TY>(a.dh, r * a.lddh + f, d);
    if constexpr (ST == T_Q8) {
      const uint8_t* q = (const uint8_t*)a.gu + r * a.ldgu + f;
      const uint8_t* sc = a.gs + r * a.ldgs + (f >> 5);
      const u32x2 qg = *(const u32x2*)q, qu = *(const u32x2*)(q + a.F);
      const float sg = q8_value(sc[0]), su = q8_value(sc[(a.F + 31) / 32]);
      q8_unpack4(qg[0], sg, g);
      q8_unpack4(qg[1], sg, g + 4);
      q8_unpack4(qu[0], su, u);
      q8_unpack4(qu[1], su, u + 4);
    } else {
      load8<TY>(a.gu, r * a.ldgu + f, g);
      load8<TY>(a.gu, r * a.ldgu + a.F + f, u);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float slope;
      const float v = act_value<true>(a.act, g[e], slope);
      h[e] = v * u[e];
      g[e] = d[e] * u[e] * slope;
      u[e] = d[e] * v;
      db[e] += g[e];
      db[8 + e] += u[e];
    }
    if (a.h) store8<TY>(a.h, r * a.ldh + f, h);
    if (a.dgu) {
      store8<TY>(a.dgu, r * a.lddgu + f, g);
      store8<TY>(a.dgu, r * a.lddgu + a.F + f, u);
    }
  }
  if (!a.part) return;  // (uniform)
#pragma unroll
  for (int e = 0; e < 16; ++e) fold[sub][e][lane] = db[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 512; i += 256) {
    const int half = i >> 8, l = (i >> 3) & 31, e = i & 7;
    const int feat = blockIdx.x * 256 + l * 8 + e;
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += fold[k][half * 8 + e][l];
    if (feat < a.F) a.part[(long long)blockIdx.y * 2 * a.F + (long long)half * a.F + feat] = t;
  }
}

// ------------------------------------------------------------------------------------------------------------- host
// Shares a product of 256 x 256 tiles out where that is shorter, in K-steps of a workgroup (1.75 us with the chip full): a
// partial tile's way to memory and back takes 0.07 of them (256 KiB twice at 4 TB/s), second jobs and launches 4.
// time: the product's, in K-steps
Share share_out(long long M, long long N, long long K, double& time) {
  Share s = {};
  s.tiles_m = (int)((M + 255) / 256);
  s.tiles_n = (int)((N + 255) / 256);
  s.steps = (int)((K + 63) / 64);
  const long long tiles = (long long)s.tiles_m * s.tiles_n;
  s.rest = (int)(tiles % 256);
  s.whole = (int)tiles;
  s.splits = 1;
  time = (double)((tiles + 255) / 256) * s.steps;
  if (s.rest == 0) return s;
  int splits = (255 + s.rest) / s.rest;
  if (splits > s.steps / 4) splits = s.steps / 4;
  if (splits < 2) return s;
  int wgs = s.rest * splits, over = 0, runs = 0;
  const double part = (double)s.steps / splits, partial = 0.07;
  double shared = part + 4;
  if (wgs > 256) {
    over = wgs - 256;
    wgs = 256;
    runs = (int)sqrt(part / (partial * over));  // part / runs + partial * over * runs at its least
    const int most = 256 / over < (int)part / 2 ? 256 / over : (int)part / 2;
    runs = runs > most ? most : runs;
    runs = runs < 1 ? 1 : runs;
    shared += part / runs;
  }
  shared += partial * (wgs + over * runs);
  if (shared > s.steps) return s;
  time = (double)(tiles / 256) * s.steps + shared;
  s.splits = splits;
  s.whole = (int)(tiles - s.rest);
  s.wgs = wgs;
  s.over = over;
  s.runs = runs;
  return s;
}

// How the backward's two products are cut: 256 x 256 tiles and a launch each, or T x T tiles with K in sx and sw parts and
// one launch for both. Counted from the sizes alone, whichever outputs are asked for: alone and together they have the
// same bits.
struct TilePlan {
  int64_t M, D, F;
  int T, sx, sw;  // T = 256: sx, sw are for strides that the 256 x 256 kernel does not reach, on 128 x 128 tiles
};
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t tiles_of(int64_t M, int64_t N, int T) { return ceil_div(M, T) * ceil_div(N, T); }

// the K-step at which the last job ends when n jobs of a steps, then m of b <= a, go to `slots` places in that order
int64_t last_end(int64_t n, int64_t a, int64_t m, int64_t b, int64_t slots) {
  const int64_t late = n % slots, early = slots - late, t0 = n / slots * a, t1 = t0 + a;  // early places are free at t0, the others at t1
  const int64_t up = ceil_div(a, b), down = a / b;
  const int64_t i = early * up >= m ? ceil_div(m, early) : ceil_div(m + late * up, slots);  // b-jobs in a row on an early place, if one ends last
  const int64_t k = m > early * down ? ceil_div(m - early * down, slots) : 0;           // on a late place
  const int64_t end = t0 + i * b < t1 + k * b ? t0 + i * b : t1 + k * b;
  return late && end < t1 ? t1 : end;
}

// The plan of least estimated time. The estimate, in us behind the element-wise part: on T x T tiles, a part for the
// K-step at which the last workgroup ends (with 512 of T = 128 or 1024 of 64 at a time), one for the mean steps of a
// place, for the MB of partials written and read, and for the splits that a sum is made of; on 256 x 256 tiles, the steps
// of share_out. Fitted to the times of 38 sizes (17 x 256 x 688 to 16384 x 768 x 2048, up to 54 plans each; 6 to 8 %
// off); the plans are 3 % behind the best measured ones on the geometric mean, at most 12 %. Equal K-steps for every
// workgroup instead, the whole backward in us: 8192 x 768 x 2048 209 to 170 here, 4096 x 512 x 1376 73 / 58,
// 4096 x 1024 x 2736 170 / 156, 1029 x 512 x 1376 37 / 29, 1029 x 256 x 688 21.7 / 20.2, 2048 x 768 x 2048 58 / 60.
// At least 4 steps a split, and no more than two rounds of jobs.
TilePlan tile_plan(int64_t M, int64_t D, int64_t F) {
  static thread_local TilePlan last = {};  // (asked for the workspace first, then for the launch)
  if (last.T && last.M == M && last.D == D && last.F == F) return last;
  TilePlan best = {M, D, F, 0, 1, 1};
  double least = 0;
  constexpr int SPLITS[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
  const int64_t kx = ceil_div(2 * F, 64), kw = ceil_div(M > 0 ? M : 1, 64);
  for (int T = 128; T >= 64; T -= 64) {
    const bool wide = T == 128;
    const int64_t slots = wide ? 512 : 1024, nx = tiles_of(M, D, T), nw = tiles_of(2 * F, D, T);
    for (int sx : SPLITS) {
      if (sx > 1 && (sx * 4 > kx || nx * sx > 2 * slots)) break;
      for (int sw : SPLITS) {
        if (sw > 1 && (sw * 4 > kw || nw * sw > 2 * slots)) break;
        const int64_t lx = ceil_div(kx, sx), lw = ceil_div(kw, sw), jx = nx * sx, jw = nw * sw;
        const int64_t end = lx >= lw ? last_end(jx, lx, jw, lw, slots) : last_end(jw, lw, jx, lx, slots);
        const double mean = (double)(jx * lx + jw * lw) / slots;
        const double mb = ((sx > 1 ? (double)sx * M * D : 0.0) + (sw > 1 ? (double)sw * 2 * F * D : 0.0)) * 8e-6;
        const int most = sx > sw ? sx : sw;
        const double us = wide ? 6.5 + 0.54 * end + 0.72 * mean + 0.13 * mb + 0.12 * most : 5.0 + 0.3 * end + 0.73 * mean + 0.135 * mb + 0.18 * most;
        if (best.T == 0 || us < least) {
          least = us;
          best.T = T;
          best.sx = sx;
          best.sw = sw;
        }
      }
    }
  }
  if (best.T == 128) {
    double x, w;
    share_out(M, D, 2 * F, x);
    share_out(2 * F, D, M, w);
    if (1.58 * (x + w) < least) best.T = 256;
  }
  last = best;
  return best;
}
TileJob tile_job(const GatedP& p, int T, int splits) {
  TileJob j = {};
  j.p = p;
  j.tiles_n = (p.N + T - 1) / T;
  j.tiles = (int)tiles_of(p.M, p.N, T);
  const int steps = (p.K + 63) / 64, len = steps > 0 ? (steps + splits - 1) / splits : 1;
  j.splits = steps > 0 ? (steps + len - 1) / len : 1;
  j.p.kper = len * 64;
  return j;
}
// its partials go to ws: what is left to do for the output that p names
JoinJob join_job(TileJob& j, void* ws) {
  JoinJob f = {};
  if (j.splits < 2) return f;
  GatedP& p = j.p;
  f.out = p.C;
  f.ldo = p.ldc;
  f.type = p.c_type;
  f.part = (const float*)ws;
  f.stride = p.split_stride = (long long)p.M * p.N;
  f.rows = p.M;
  f.nch = p.N / 8;
  f.splits = j.splits;
  f.blocks = (unsigned)((f.rows * f.nch + 255) / 256);
  p.C = ws;
  p.ldc = p.N;
  p.c_type = T_F32;
  return f;
}

template <int TY, int MODE>
int product_big(const GatedP& p, const Share& sh, void* ws, hipStream_t s) {
  (void)hipFuncSetAttribute((const void*)gated_big_kernel<TY, MODE>, hipFuncAttributeMaxDynamicSharedMemorySize, 2 * STAGE);
  hipLaunchKernelGGL((gated_big_kernel<TY, MODE>), dim3((unsigned)(sh.whole + sh.wgs)), dim3(512), 2 * STAGE, s, p, sh, (float*)ws);
  if (sh.wgs)
    hipLaunchKernelGGL((gated_fix_kernel<TY>), dim3(32, (unsigned)sh.rest), dim3(256), 0, s, p, sh, (const float*)ws);
  return 0;
}
// operand strides up to which the 256 x 256 kernel's 32-bit offsets reach
bool near(int64_t ld) { return ld < (1 << 21); }

template <int TY>
int forward(const GatedP& p, hipStream_t s) {
  // Up to 16 rows, and up to 64 where the 16-feature workgroups are at most one for each CU (8-bit saves, 32 features a
  // workgroup: 32). Measured against the tiles (bf16, us): 32 x 1280 x 3416 7.2 / 11.2, 64 x 1024 x 4096 8.4 / 9.9,
  // 64 x 1280 x 3416 9.6 / 11.3, 64 x 256 x 688 3.7 / 4.0, but 64 x 1024 x 5504 13.6 / 9.9, 32 x 4096 x 11008 45 / 39
  const bool few = p.N <= 16 * 256;
  if (p.M <= 16 || (few && p.M <= (p.save_type == T_Q8 ? 32 : 64))) {
    if (p.M <= 16) forward_few<TY, 1>(p, s);
    else if (p.M <= 32) forward_few<TY, 2>(p, s);
    else forward_few16<TY, 4>(p, s);
    return 0;
  }
  // The tile: 128 rows x 128 features once its tiles fill most of the 256 CUs, 128 x 64 once those fill them, else 64 x 32.
  // Measured (bf16, us): 2048 x 1024 x 2736 28 / 38 / 51, 1024 x 1280 x 3416 (216 large tiles) 29.1 / 30.6 / 48,
  // 4096 x 256 x 688 (192) 10.6 / 9.8 / 11.2, 512 x 1280 x 3416 (108, 216) 27 / 22.5 / 29, 512 x 768 x 2048 (64, 128)
  // - / 13.8 / 10.5
  const int64_t duo_m = ((int64_t)p.M + 127) / 128, duo_n = ((int64_t)p.N + 127) / 128;
  OCTSAM_CHECK_ARG(duo_m * duo_n < (1 << 26), "gated_fwd: too many tiles");
  if (duo_m * duo_n >= 200 && near(p.lda) && near(p.ldb)) {
    (void)hipFuncSetAttribute((const void*)gated_duo_kernel<TY>, hipFuncAttributeMaxDynamicSharedMemorySize, DUO_LDS);
    hipLaunchKernelGGL((gated_duo_kernel<TY>), dim3((unsigned)(duo_m * duo_n)), dim3(256), DUO_LDS, s, p, (int)duo_m, (int)duo_n);
    return 0;
  }
  GatedP q = p;
  q.kper = (p.K + 63) / 64 * 64;
  const int64_t large = ((int64_t)p.M + 127) / 128 * (((int64_t)p.N + 63) / 64), small = ((int64_t)p.M + 63) / 64 * (((int64_t)p.N + 31) / 32);
  if (large >= 192)
    hipLaunchKernelGGL((gated_tile_kernel<TY, 128>), dim3((unsigned)large), dim3(256), 0, s, q, (p.N + 63) / 64);
  else
    hipLaunchKernelGGL((gated_tile_kernel<TY, 64>), dim3((unsigned)small), dim3(256), 0, s, q, (p.N + 31) / 32);
  return 0;
}

int64_t round16(int64_t n) { return (n + 15) & ~(int64_t)15; }
// bytes of fp32 partials of a product
int64_t partial_bytes(int64_t M, int64_t N, int64_t K, int T, int most) {
  if (M <= 0 || N <= 0) return 0;
  double time;
  const Share sh = share_out(M, N, K, time);
  const int64_t big = T == 256 ? (int64_t)(sh.wgs + sh.over * sh.runs) * 65536 * 4 : 0;
  GatedP p = {};
  p.M = (int)M;
  p.N = (int)N;
  p.K = (int)K;
  const int splits = tile_job(p, T == 64 ? 64 : 128, most).splits;
  const int64_t small = splits > 1 ? splits * M * N * 4 : 0;
  return round16(big > small ? big : small);
}

// rows per workgroup of the element-wise backward (grid y: at most 32768 workgroups)
int64_t slab_of(int64_t M) {
  const int64_t least = (M + 32767) / 32768, want = M <= 2048 ? 8 : 32;
  return least > want ? (least + 7) / 8 * 8 : want;
}

struct BwdPlan {
  int64_t dgu, x16, part, join_x, join_w, total;
  TilePlan tiles;
  int64_t slab;
  int slabs;
};
BwdPlan bwd_plan(int64_t M, int64_t D, int64_t F, bool x_q8) {
  BwdPlan b;
  b.slab = slab_of(M);
  b.slabs = (int)((M + b.slab - 1) / b.slab);
  int64_t at = 0;
  b.dgu = at;
  at += round16(M * 2 * F * 2);
  b.x16 = at;
  at += x_q8 ? round16(M * D * 2) : 0;
  b.part = at;
  at += round16((int64_t)b.slabs * 2 * F * 4);
  b.join_x = at;
  b.tiles = tile_plan(M, D, F);
  at += partial_bytes(M, D, 2 * F, b.tiles.T, b.tiles.sx);
  b.join_w = at;
  at += partial_bytes(2 * F, D, M, b.tiles.T, b.tiles.sw);
  b.total = at;
  return b;
}

bool row_ok(const void* p, int64_t ld, int bytes) { return !p || (ld % 8 == 0 && aligned(p, bytes)); }
constexpr int64_t MAX_M = 1ll << 30, MAX_W = 1 << 24;

template <int TY>
int run_bwd(const BwdPlan& b, const ActBwd& act, int gu_type, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M,
            int D, int F, void* dx, int64_t lddx, void* dw, int dw_type, int64_t lddw, float* db, char* ws, hipStream_t s) {
  if (M > 0) {
    const dim3 grid((unsigned)((F + 255) / 256 + (act.x8 ? (D + 255) / 256 : 0)), (unsigned)b.slabs);
    if (gu_type == T_Q8) hipLaunchKernelGGL((gated_act_bwd_kernel<TY, T_Q8>), grid, dim3(256), 0, s, act);
    else hipLaunchKernelGGL((gated_act_bwd_kernel<TY, TY>), grid, dim3(256), 0, s, act);
  }
  GatedP px = {}, pw = {};
  px.A = pw.A = ws + b.dgu;
  px.lda = pw.lda = 2 * (int64_t)F;
  px.save_type = pw.save_type = T_NONE;
  px.N = pw.N = D;
  px.B = w, px.ldb = ldw, px.C = dx, px.ldc = lddx, px.c_type = TY, px.M = (int)M, px.K = 2 * F;
  pw.B = x, pw.ldb = ldx, pw.C = dw, pw.ldc = lddw, pw.c_type = dw_type, pw.M = 2 * F, pw.K = (int)M;
  double time;
  const Share shx = share_out(M, D, 2 * F, time), shw = share_out(2 * F, D, M, time);
  const bool big = b.tiles.T == 256 && near(px.lda), big_x = big && near(ldw), big_w = big && M > 0 && near(ldx);
  if (dx && M > 0 && big_x)
    if (int rc = product_big<TY, NN>(px, shx, ws + b.join_x, s)) return rc;
  if (dw && big_w)
    if (int rc = product_big<TY, TN>(pw, shw, ws + b.join_w, s)) return rc;
  const bool tile_x = dx && M > 0 && !big_x, tile_w = dw && !big_w;
  TileJob jx = {}, jw = {};
  JoinJob fx = {}, fw = {};
  if (tile_x || tile_w) {
    const int T = b.tiles.T == 64 ? 64 : 128;
    OCTSAM_CHECK_ARG(tiles_of(M, D, T) + tiles_of(2 * F, D, T) < (1 << 24), "gated_bwd: too many tiles");
    if (tile_x) jx = tile_job(px, T, b.tiles.sx), fx = join_job(jx, ws + b.join_x);
    if (tile_w) jw = tile_job(pw, T, b.tiles.sw), fw = join_job(jw, ws + b.join_w);
    const int blocks = jx.tiles * jx.splits + jw.tiles * jw.splits;
    const bool w_first = jw.p.kper > jx.p.kper;
    if (T == 64) hipLaunchKernelGGL((gated_pair_kernel<TY, 64>), dim3((unsigned)blocks), dim3(256), 0, s, jx, jw, w_first);
    else hipLaunchKernelGGL((gated_pair_kernel<TY, 128>), dim3((unsigned)blocks), dim3(256), 0, s, jx, jw, w_first);
  }
  DbJob d = {};
  if (db) {
    d.part = (const float*)(ws + b.part);
    d.out = db;
    d.slabs = b.slabs;  // (none without rows: db is zero)
    d.n = 2 * F;
    d.blocks = (unsigned)((d.n + SUM_COLS - 1) / SUM_COLS);
  }
  if (const unsigned blocks = fx.blocks + fw.blocks + d.blocks)
    hipLaunchKernelGGL((gated_finish_kernel<TY>), dim3(blocks), dim3(256), 0, s, fx, fw, d);
  return 0;
}

}  // namespace

extern "C" int octsam_gated_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const float* bias, int64_t M, int32_t D,
                                int32_t F, int32_t act, int32_t type, void* h, int64_t ldh, void* save, int32_t save_type,
                                int64_t ld_save, void* save_scale, int64_t ld_scale, void* stream) {
  OCTSAM_CHECK_ARG(type == T_BF16 || type == T_F16, "gated_fwd: operands are bf16 or fp16");
  OCTSAM_CHECK_ARG(act >= 0 && act <= OCTSAM_ACT_SILU, "gated_fwd: unknown activation %d", act);
  OCTSAM_CHECK_ARG(M >= 0 && M <= MAX_M && D > 0 && D <= MAX_W && F > 0 && F <= MAX_W, "gated_fwd: M %lld, D %d, F %d",
                   (long long)M, D, F);
  OCTSAM_CHECK_ARG(D % 8 == 0 && F % 8 == 0, "gated_fwd: D and F are multiples of 8 (16-byte rows), got %d and %d", D, F);
  if (M == 0) return 0;
  OCTSAM_CHECK_ARG(x && w && h, "gated_fwd: null operand");
  OCTSAM_CHECK_ARG(!save || save_type == type || save_type == T_Q8, "gated_fwd: save is of the operands' type or 8-bit");
  OCTSAM_CHECK_ARG((save && save_type == T_Q8) == (save_scale != nullptr), "gated_fwd: scales come with an 8-bit save, and only with it");
  OCTSAM_CHECK_ARG(ldx >= D && ldw >= D && ldh >= F && (!save || ld_save >= 2 * (int64_t)F) &&
                       (!save_scale || ld_scale >= 2 * ((F + 31) / 32)),
                   "gated_fwd: a row stride is below the row's width");
  OCTSAM_CHECK_ARG(row_ok(x, ldx, 16) && row_ok(w, ldw, 16) && row_ok(h, ldh, 16) &&
                       row_ok(save, ld_save, save_type == T_Q8 ? 8 : 16) && aligned(bias, 16),
                   "gated_fwd: rows start at multiples of 16 bytes (8 for an 8-bit save)");
  GatedP p = {};
  p.A = x;
  p.lda = ldx;
  p.B = w;
  p.ldb = ldw;
  p.bias = bias;
  p.C = h;
  p.ldc = ldh;
  p.save = save;
  p.save_type = save ? save_type : T_NONE;
  p.scale = (uint8_t*)save_scale;
  p.ldsave = ld_save;
  p.ldscale = ld_scale;
  p.M = (int)M;
  p.N = F;
  p.K = D;
  p.act = act;
  const int rc = type == T_BF16 ? forward<T_BF16>(p, (hipStream_t)stream) : forward<T_F16>(p, (hipStream_t)stream);
  if (rc) return rc;
  OCTSAM_LAUNCH_CHECK("octsam_gated_fwd");
  return 0;
}

extern "C" int64_t octsam_gated_bwd_workspace(int64_t M, int32_t D, int32_t F, int32_t x_q8) {
  if (M < 0 || M > MAX_M || D <= 0 || D > MAX_W || F <= 0 || F > MAX_W) return 0;
  return bwd_plan(M, D, F, x_q8 != 0).total;
}

extern "C" int octsam_gated_bwd(const void* dh, int64_t lddh, const void* gu, int32_t gu_type, int64_t ldgu, const void* gu_scale,
                                int64_t ld_gu_scale, const void* x, int32_t x_type, int64_t ldx, const void* x_scale,
                                int64_t ld_x_scale, const void* w, int64_t ldw, int64_t M, int32_t D, int32_t F, int32_t act,
                                int32_t type, void* h, int64_t ldh, void* dx, int64_t lddx, void* dw, int32_t dw_type,
                                int64_t lddw, float* db, void* workspace, int64_t workspace_bytes, void* stream) {
  OCTSAM_CHECK_ARG(type == T_BF16 || type == T_F16, "gated_bwd: operands are bf16 or fp16");
  OCTSAM_CHECK_ARG(act >= 0 && act <= OCTSAM_ACT_SILU, "gated_bwd: unknown activation %d", act);
  OCTSAM_CHECK_ARG(M >= 0 && M <= MAX_M && D > 0 && D <= MAX_W && F > 0 && F <= MAX_W, "gated_bwd: M %lld, D %d, F %d",
                   (long long)M, D, F);
  OCTSAM_CHECK_ARG(D % 8 == 0 && F % 8 == 0, "gated_bwd: D and F are multiples of 8 (16-byte rows), got %d and %d", D, F);
  OCTSAM_CHECK_ARG(M == 0 || h || dx || dw || db, "gated_bwd: no output");  // (an empty output has no address)
  OCTSAM_CHECK_ARG(M == 0 || (dh && gu), "gated_bwd: null operand");
  OCTSAM_CHECK_ARG(gu_type == type || gu_type == T_Q8, "gated_bwd: the kept projections are of the operands' type or 8-bit");
  OCTSAM_CHECK_ARG(M == 0 || (gu_type == T_Q8) == (gu_scale != nullptr), "gated_bwd: scales come with 8-bit projections, and only with them");
  OCTSAM_CHECK_ARG(!dx || M == 0 || w, "gated_bwd: dx needs w");
  OCTSAM_CHECK_ARG(!dw || dw_type == type || dw_type == T_F32, "gated_bwd: dw is fp32 or of the operands' type");
  const bool xq = dw && x_type == T_Q8;
  OCTSAM_CHECK_ARG(!dw || ((x || M == 0) && (x_type == type || (x_type == T_Q8 && (x_scale || M == 0)))),
                   "gated_bwd: dw needs x, of the operands' type or 8-bit with its scales");
  OCTSAM_CHECK_ARG(lddh >= F && ldgu >= 2 * (int64_t)F && (gu_type != T_Q8 || ld_gu_scale >= 2 * ((F + 31) / 32)) &&
                       (!dw || ldx >= D) && (!xq || ld_x_scale >= (D + 31) / 32) && (!dx || (ldw >= D && lddx >= D)) &&
                       (!h || ldh >= F) && (!dw || lddw >= D),
                   "gated_bwd: a row stride is below the row's width");
  OCTSAM_CHECK_ARG(row_ok(dh, lddh, 16) && row_ok(gu, ldgu, gu_type == T_Q8 ? 8 : 16) && (!dw || row_ok(x, ldx, xq ? 8 : 16)) &&
                       (!dx || (row_ok(w, ldw, 16) && row_ok(dx, lddx, 16))) && row_ok(h, ldh, 16) && row_ok(dw, lddw, 16) &&
                       aligned(db, 4),
                   "gated_bwd: rows start at multiples of 16 bytes (8 for 8-bit operands)");
  const BwdPlan b = bwd_plan(M, D, F, xq);
  OCTSAM_CHECK_ARG(workspace && aligned(workspace, 16) && workspace_bytes >= b.total,
                   "gated_bwd: the workspace needs %lld bytes, 16-B aligned", (long long)b.total);
  const hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  ActBwd a = {};
  a.dh = dh, a.lddh = lddh, a.gu = gu, a.ldgu = ldgu, a.gs = (const uint8_t*)gu_scale, a.ldgs = ld_gu_scale;
  a.dgu = dx || dw ? ws + b.dgu : nullptr, a.lddgu = 2 * (int64_t)F;
  a.h = h, a.ldh = ldh, a.part = db ? (float*)(ws + b.part) : nullptr;
  a.M = M, a.F = F, a.act = act, a.slab = b.slab;
  if (xq) {
    a.x8 = x, a.ldx = ldx, a.xs = (const uint8_t*)x_scale, a.ldxs = ld_x_scale, a.D = D;
    x = a.x16 = ws + b.x16;
    ldx = D;
  }
  const int rc = type == T_BF16 ? run_bwd<T_BF16>(b, a, gu_type, x, ldx, w, ldw, M, D, F, dx, lddx, dw, dw_type, lddw, db, ws, s)
                                : run_bwd<T_F16>(b, a, gu_type, x, ldx, w, ldw, M, D, F, dx, lddx, dw, dw_type, lddw, db, ws, s);
  if (rc) return rc;
  OCTSAM_LAUNCH_CHECK("octsam_gated_bwd");
  return 0;
}
