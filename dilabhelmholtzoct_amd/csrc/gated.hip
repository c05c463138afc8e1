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
// Tile: 64 x 64 x 64, four waves of 16 rows x 64 columns of 16x16x32 MFMAs with swapped operands (a lane holds 4
// consecutive columns of a row; one permlane16_swap makes 8). In the forward the 64 columns are 32 gate rows and the 32
// up rows of the same features, so a lane has g and u of the same 8 features and four lanes hold an 8-bit group.
// Operands with k contiguous and operands stored [k][x] (W in dx, both in dW) use the same loop: the second kind is
// read from LDS with the transposing 64-bit read. Global loads run three K-steps ahead in registers.
#include "q8.h"
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

// act(g) and, with GRAD, act'(g)
template <bool GRAD>
__device__ __forceinline__ float act_value(int act, float g, float& slope) {
  if (act == OCT_SILU) {
    const float p = 1.0f / (1.0f + __expf(-g));
    if constexpr (GRAD) slope = p * fmaf(g, 1.0f - p, 1.0f);
    return g * p;
  }
  if (act == OCT_GELU) {
    const float cdf = 0.5f * (1.0f + erf_fast(g * 0.70710678118654752f));
    if constexpr (GRAD) slope = fmaf(g * 0.3989422804014327f, __expf(-0.5f * g * g), cdf);
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

__device__ __forceinline__ void keep8_q(const GatedP& p, long long m, int half, int f, bool ok, const float* v) {
  float a = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) a = fmaxf(a, ok ? finite_abs(v[e]) : 0.0f);
  a = fmaxf(a, __shfl_xor(a, 16, 64));
  a = fmaxf(a, __shfl_xor(a, 32, 64));
  if (ok) {
    const int b = q8_scale(a);
    const float inv = q8_inverse(b);
    *(u32x2*)((uint8_t*)p.save + m * p.ldsave + (long long)half * p.N + f) = (u32x2){q8_pack4(v, inv), q8_pack4(v + 4, inv)};
    if ((f & 31) == 0) p.scale[m * p.ldscale + half * ((p.N + 31) / 32) + (f >> 5)] = (uint8_t)b;
  }
}

// g, u: a lane's 8 features from f on of row m (all lanes of a wave call this together). Rows past M and features
// past F (a multiple of 8) are dropped; f % 32 is the same in the four lanes that hold an 8-bit group
template <int TY>
__device__ __forceinline__ void gated_store(const GatedP& p, long long m, int f, float* g, float* u) {
  const bool ok = m < p.M && f < p.N;
  if (p.bias && ok) {
    float b[8];
    load8<T_F32>(p.bias, f, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] += b[e];
    load8<T_F32>(p.bias, (long long)p.N + f, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] += b[e];
  }
  if (p.save_type == T_Q8) {
    keep8_q(p, m, 0, f, ok, g);
    keep8_q(p, m, 1, f, ok, u);
  } else if (p.save_type != T_NONE && ok) {
    store8<TY>(p.save, m * p.ldsave + f, g);
    store8<TY>(p.save, m * p.ldsave + p.N + f, u);
  }
  if (ok) {
    float h[8], unused;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = act_value<false>(p.act, g[e], unused) * u[e];
    store8<TY>(p.C, m * p.ldc + f, h);
  }
}

template <int TY>
__device__ __forceinline__ void plain_store(const GatedP& p, long long m, int n, int split, const float* v) {
  if (m >= p.M || n >= p.N) return;
  const long long at = m * p.ldc + n;
  if (p.c_type == T_F32) store8<T_F32>((float*)p.C + split * p.split_stride, at, v);
  else store8<TY>(p.C, at, v);
}

// ------------------------------------------------------------------------------------------------------- 64 x 64 tile
// LDS images [64 rows][128 B]; 16-B chunk c of row r sits at c ^ swizzle. Rows of k (KC): (r >> 1) & 7, the 16 rows of
// a fragment read land on 16 slots. [k][x] (KM): the four rows q of a 16-lane group and the group pair (r bit 3) land
// on 8 slot pairs of two rows.
__device__ __forceinline__ int kc_at(int r, int c) { return r * 128 + ((c ^ ((r >> 1) & 7)) << 4); }
__device__ __forceinline__ int km_at(int r, int c) { return r * 128 + ((c ^ ((r & 2) | ((r >> 1) & 4))) << 4); }

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <int TY, bool KM>
__device__ __forceinline__ typename Elem<TY>::v8 frag64(const char* img, int x0, int kb, int lane) {
  typedef typename Elem<TY>::v8 v8;
  if constexpr (!KM) {
    return *(const v8*)(img + kc_at(x0 + (lane & 15), kb * 4 + (lane >> 4)));
  } else {
    const int g = lane >> 4, i = lane & 15, q = i >> 2, pp = i & 3;
    const char* at = img + km_at(kb * 32 + 8 * g + q, (x0 >> 3) + (pp >> 1)) + 8 * (pp & 1);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 4 * 128));  // (+4 leaves the swizzle)
    const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(v8, v);
  }
}

template <int TY, int MODE>
__global__ __launch_bounds__(256) void gated_tile_kernel(GatedP p, int tiles_n) {
  typedef typename Elem<TY>::v8 v8;
  constexpr bool AKM = MODE == TN, BKM = MODE != GATED;
  constexpr int AHEAD = 3, IMG = 64 * 128;
  __shared__ __attribute__((aligned(16))) char smem[2][2][IMG];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tm = blockIdx.x / tiles_n, tn = blockIdx.x - tm * tiles_n;
  const long long row0 = (long long)tm * 64;
  const int col0 = tn * (MODE == GATED ? 32 : 64);
  const long long k0 = (long long)blockIdx.y * p.kper;
  const int kn = (int)(p.K - k0 < p.kper ? p.K - k0 : p.kper);  // (< 1: no steps, the tile is zero)
  const int steps = kn > 0 ? (kn + 63) / 64 : 0;

  // this thread's two 16-B pieces of each operand's stage: image row rr (and rr + 32), chunk cc
  const int rr = tid >> 3, cc = tid & 7;
  const char *pa[2], *pb[2];
  bool oa[2], ob[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = rr + 32 * i;
    if constexpr (AKM) {
      oa[i] = row0 + cc * 8 < p.M;
      pa[i] = (const char*)p.A + ((k0 + r) * p.lda + row0 + cc * 8) * 2;
    } else {
      oa[i] = row0 + r < p.M;
      pa[i] = (const char*)p.A + ((row0 + r) * p.lda + k0 + cc * 8) * 2;
    }
    if constexpr (BKM) {
      ob[i] = col0 + cc * 8 < p.N;
      pb[i] = (const char*)p.B + ((k0 + r) * p.ldb + col0 + cc * 8) * 2;
    } else {
      ob[i] = col0 + rr < p.N;  // image rows 0-31: gate features, 32-63: the same features' up rows
      pb[i] = (const char*)p.B + (((long long)i * p.N + col0 + rr) * p.ldb + k0 + cc * 8) * 2;
    }
  }
  const long long sa = AKM ? p.lda * 128 : 128, sb = BKM ? p.ldb * 128 : 128;
  u32x4 ra[AHEAD][2], rb[AHEAD][2];
  auto fetch = [&](int t, u32x4 (&a)[2], u32x4 (&b)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int ka = t * 64 + (AKM ? rr + 32 * i : cc * 8), kb = t * 64 + (BKM ? rr + 32 * i : cc * 8);
      a[i] = oa[i] && ka < kn ? *(const u32x4*)(pa[i] + t * sa) : (u32x4)0u;
      b[i] = ob[i] && kb < kn ? *(const u32x4*)(pb[i] + t * sb) : (u32x4)0u;
    }
  };
#pragma unroll
  for (int j = 0; j < AHEAD; ++j)
    if (j < steps) fetch(j, ra[j], rb[j]);
  f32x4 acc[4] = {(f32x4)0.0f, (f32x4)0.0f, (f32x4)0.0f, (f32x4)0.0f};
  for (int t0 = 0; t0 < steps; t0 += AHEAD) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int t = t0 + j;
      if (t < steps) {
        char *ia = smem[t & 1][0], *ib = smem[t & 1][1];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          *(u32x4*)(ia + (AKM ? km_at(rr + 32 * i, cc) : kc_at(rr + 32 * i, cc))) = ra[j][i];
          *(u32x4*)(ib + (BKM ? km_at(rr + 32 * i, cc) : kc_at(rr + 32 * i, cc))) = rb[j][i];
        }
        if (t + AHEAD < steps) fetch(t + AHEAD, ra[j], rb[j]);
        // one barrier a step: whoever writes this buffer again has passed the next step's barrier, and so have all
        // its readers of this step
        __syncthreads();
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const v8 af = frag64<TY, AKM>(ia, wave * 16, kb, lane);
#pragma unroll
          for (int ni = 0; ni < 4; ++ni) acc[ni] = mma<TY>(frag64<TY, BKM>(ib, ni * 16, kb, lane), af, acc[ni]);
        }
      }
    }
  }
  const int q = lane >> 4, cofs = 16 * (q & 1) + 8 * (q >> 1);
  const long long m = row0 + wave * 16 + (lane & 15);
  float v0[8], v1[8];
  row8(acc[0], acc[1], v0);
  row8(acc[2], acc[3], v1);
  if constexpr (MODE == GATED) {
    gated_store<TY>(p, m, col0 + cofs, v0, v1);
  } else {
    plain_store<TY>(p, m, col0 + cofs, blockIdx.y, v0);
    plain_store<TY>(p, m, col0 + 32 + cofs, blockIdx.y, v1);
  }
}

// out = the sum of the K splits' fp32 partials in order, rounded once
template <int TY>
__global__ __launch_bounds__(256) void gated_join_kernel(const float* __restrict__ part, long long stride, int splits,
                                                         long long rows, int nch, void* __restrict__ out, long long ldo) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * nch) return;
  const long long r = i / nch;
  float v[8], t[8];
  load8<T_F32>(part, i * 8, v);
  for (int s = 1; s < splits; ++s) {
    load8<T_F32>(part, s * stride + i * 8, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += t[e];
  }
  store8<TY>(out, r * ldo + (i - r * nch) * 8, v);
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
};

// workgroup (x, y): 256 features (32 lanes of 8) of the rows [y * slab, (y + 1) * slab), eight rows at a time
template <int TY, int ST>
__global__ __launch_bounds__(256) void gated_act_bwd_kernel(ActBwd a) {
  __shared__ float fold[8][16][33];
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
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

__global__ void gated_zero_kernel(float* p, long long n) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = 0.0f;
}

// ------------------------------------------------------------------------------------------------------------- host
// K splits of a product with `tiles` output tiles: enough workgroups for the chip's 256 CUs twice over, at least four
// K-steps each
int splits_for(long long tiles, long long K) {
  const long long steps = (K + 63) / 64, want = (511 + tiles) / tiles, most = steps / 4;
  const long long s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}
int kper_of(long long K, int splits) { return (int)(((K + 63) / 64 + splits - 1) / splits * 64); }

template <int TY, int MODE>
int product(GatedP p, void* ws, hipStream_t s) {
  const long long tiles_m = ((long long)p.M + 63) / 64, tiles_n = MODE == GATED ? ((long long)p.N + 31) / 32 : ((long long)p.N + 63) / 64;
  const long long tiles = tiles_m * tiles_n;
  OCTSAM_CHECK_ARG(tiles < (1ll << 31), "gated: too many tiles");
  if (MODE == GATED) {
    p.kper = (p.K + 63) / 64 * 64;
    hipLaunchKernelGGL((gated_tile_kernel<TY, MODE>), dim3((unsigned)tiles), dim3(256), 0, s, p, (int)tiles_n);
    return 0;
  }
  const int splits = splits_for(tiles, p.K);
  p.kper = kper_of(p.K, splits);
  if (splits == 1) {
    hipLaunchKernelGGL((gated_tile_kernel<TY, MODE>), dim3((unsigned)tiles), dim3(256), 0, s, p, (int)tiles_n);
    return 0;
  }
  void* out = p.C;
  const long long ldo = p.ldc;
  const int out_type = p.c_type;
  p.C = ws;
  p.ldc = p.N;
  p.c_type = T_F32;
  p.split_stride = (long long)p.M * p.N;
  hipLaunchKernelGGL((gated_tile_kernel<TY, MODE>), dim3((unsigned)tiles, splits), dim3(256), 0, s, p, (int)tiles_n);
  const long long items = (long long)p.M * (p.N / 8);
  if (out_type == T_F32)
    hipLaunchKernelGGL((gated_join_kernel<T_F32>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s, (const float*)ws,
                       p.split_stride, splits, (long long)p.M, p.N / 8, out, ldo);
  else
    hipLaunchKernelGGL((gated_join_kernel<TY>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s, (const float*)ws,
                       p.split_stride, splits, (long long)p.M, p.N / 8, out, ldo);
  return 0;
}

int64_t round16(int64_t n) { return (n + 15) & ~(int64_t)15; }
int64_t join_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0) return 0;
  const int s = splits_for(((M + 63) / 64) * ((N + 63) / 64), K);
  return s > 1 ? s * M * N * 4 : 0;
}
// rows per workgroup of the element-wise backward (grid y: at most 32768 workgroups)
int64_t slab_of(int64_t M) {
  const int64_t least = (M + 32767) / 32768, want = M <= 64 ? 8 : M <= 2048 ? 32 : 64;
  return least > want ? (least + 7) / 8 * 8 : want;
}

struct BwdPlan {
  int64_t dgu, x16, part, join, total;
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
  b.join = at;
  const int64_t j1 = join_bytes(M, D, 2 * F), j2 = join_bytes(2 * F, D, M);
  at += round16(j1 > j2 ? j1 : j2);
  b.total = at;
  return b;
}

bool row_ok(const void* p, int64_t ld, int bytes) { return !p || (ld % 8 == 0 && aligned(p, bytes)); }
constexpr int64_t MAX_M = 1ll << 30, MAX_W = 1 << 24;

template <int TY>
int run_bwd(const BwdPlan& b, const ActBwd& act, int gu_type, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M,
            int D, int F, void* dx, int64_t lddx, void* dw, int dw_type, int64_t lddw, char* ws, hipStream_t s) {
  if (M > 0) {
    const dim3 grid((unsigned)((F + 255) / 256), (unsigned)b.slabs);
    if (gu_type == T_Q8) hipLaunchKernelGGL((gated_act_bwd_kernel<TY, T_Q8>), grid, dim3(256), 0, s, act);
    else hipLaunchKernelGGL((gated_act_bwd_kernel<TY, TY>), grid, dim3(256), 0, s, act);
  }
  GatedP p = {};
  p.save_type = T_NONE;
  if (dx && M > 0) {
    p.A = ws + b.dgu;
    p.lda = 2 * (int64_t)F;
    p.B = w;
    p.ldb = ldw;
    p.C = dx;
    p.ldc = lddx;
    p.c_type = TY;
    p.M = (int)M;
    p.N = D;
    p.K = 2 * F;
    if (int rc = product<TY, NN>(p, ws + b.join, s)) return rc;
  }
  if (dw) {
    p.A = ws + b.dgu;
    p.lda = 2 * (int64_t)F;
    p.B = x;
    p.ldb = ldx;
    p.C = dw;
    p.ldc = lddw;
    p.c_type = dw_type;
    p.M = 2 * F;
    p.N = D;
    p.K = (int)M;
    if (int rc = product<TY, TN>(p, ws + b.join, s)) return rc;
  }
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
  const int rc = type == T_BF16 ? product<T_BF16, GATED>(p, nullptr, (hipStream_t)stream)
                                : product<T_F16, GATED>(p, nullptr, (hipStream_t)stream);
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
  const ActBwd a = {dh, gu, (const uint8_t*)gu_scale, dx || dw ? ws + b.dgu : nullptr, h, db ? (float*)(ws + b.part) : nullptr,
                    lddh, ldgu, ld_gu_scale, 2 * (int64_t)F, ldh, M, b.slab, F, act};
  if (xq && M > 0) {
    if (int rc = octsam_dequant8(x, ldx, x_scale, ld_x_scale, M, D, ws + b.x16, type, D, stream)) return rc;
    x = ws + b.x16;
    ldx = D;
  }
  const int rc = type == T_BF16 ? run_bwd<T_BF16>(b, a, gu_type, x, ldx, w, ldw, M, D, F, dx, lddx, dw, dw_type, lddw, ws, s)
                                : run_bwd<T_F16>(b, a, gu_type, x, ldx, w, ldw, M, D, F, dx, lddx, dw, dw_type, lddw, ws, s);
  if (rc) return rc;
  OCTSAM_LAUNCH_CHECK("octsam_gated_bwd");
  if (!db) return 0;
  if (M == 0) {
    hipLaunchKernelGGL(gated_zero_kernel, dim3((unsigned)((2ll * F + 255) / 256)), dim3(256), 0, s, db, 2ll * F);
    OCTSAM_LAUNCH_CHECK("octsam_gated_bwd");
    return 0;
  }
  return octsam_splitk_reduce((const float*)(ws + b.part), db, 2 * (int64_t)F, b.slabs, 0.0f, stream);
}
