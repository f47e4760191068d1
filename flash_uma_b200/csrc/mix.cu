// Per-system weights of a mixture of linear experts and their gradients. With a system's E coefficients
// c[s, :] and the expert matrices X[e, :] (P elements each, in any shape):
//
//   W[s, p]   = sum_e c[s, e] X[e, p]
//   dX[e, p]  = sum_s c[s, e] dW[s, p]      (the same map with c transposed)
//   dc[s, e]  = sum_p dW[s, p] X[e, p]
//
// Coefficients and their gradients are fp32, the matrices fp32, bf16 or fp16; sums are fp32, and the sum over
// P is joined in fp64.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include <cuda.h>

#include "common.cuh"
#include "grouped.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace fuma {

namespace {

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (__is_same(T, __nv_bfloat16)) return __bfloat162float(v);
  else return __half2float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (__is_same(T, __nv_bfloat16)) return __float2bfloat16_rn(v);
  else return __float2half_rn(v);
}

// Columns [p, p + 4) of a row, zeros behind the end. kVec: rows are aligned for 4-element loads.
template <typename T, bool kVec>
__device__ __forceinline__ float4 load4(const T* row, int64_t p, int64_t P) {
  if constexpr (kVec) {
    if (p >= P) return f4(0.0f);
    if constexpr (sizeof(T) == 4) {
      return *reinterpret_cast<const float4*>(row + p);
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(row + p);
      T h[4];
      memcpy(h, &u, 8);
      return make_float4(to_f32(h[0]), to_f32(h[1]), to_f32(h[2]), to_f32(h[3]));
    }
  } else {
    return make_float4(p < P ? to_f32(row[p]) : 0.f, p + 1 < P ? to_f32(row[p + 1]) : 0.f,
                       p + 2 < P ? to_f32(row[p + 2]) : 0.f, p + 3 < P ? to_f32(row[p + 3]) : 0.f);
  }
}
template <typename T, bool kVec>
__device__ __forceinline__ void store4(T* row, int64_t p, int64_t P, float4 v) {
  if constexpr (kVec) {
    if (p >= P) return;
    if constexpr (sizeof(T) == 4) {
      st4_stream(row + p, v);
    } else {
      T h[4] = {from_f32<T>(v.x), from_f32<T>(v.y), from_f32<T>(v.z), from_f32<T>(v.w)};
      uint2 u;
      memcpy(&u, h, 8);
      __stcs(reinterpret_cast<uint2*>(row + p), u);
    }
  } else {
    if (p < P) row[p] = from_f32<T>(v.x);
    if (p + 1 < P) row[p + 1] = from_f32<T>(v.y);
    if (p + 2 < P) row[p + 2] = from_f32<T>(v.z);
    if (p + 3 < P) row[p + 3] = from_f32<T>(v.w);
  }
}

constexpr int kMixCols = 256, kMixRows = 32, kMixE = 64;
constexpr int kMixSmem = kMixE * (kMixCols + kMixRows) * 4;

}  // namespace

// out[s, p] = sum_e c[s, e] X[e, p]: a block holds 256 columns of up to 64 matrices in shared memory (read
// once when there are at most 64) and goes over the rows s in tiles of 32: a thread has 8 rows x
// 4 columns, three 16-byte shared loads per 32 products.
template <typename T, bool kVec>
__global__ void __launch_bounds__(256) mix_kernel(const float* __restrict__ c, int64_t cs, int64_t ce,
                                                  const T* __restrict__ X, int S, int E, int64_t P,
                                                  T* __restrict__ out) {
  extern __shared__ float sm[];
  float* xs = sm;                      // [kMixE][kMixCols]
  float* cf = sm + kMixE * kMixCols;   // [kMixE][kMixRows]
  const int col = (threadIdx.x & 63) * 4, rg = threadIdx.x >> 6;
  const int64_t p0 = (int64_t)blockIdx.x * kMixCols;
  const int echunks = (E + kMixE - 1) / kMixE;
  for (int s0 = 0; s0 < S; s0 += kMixRows) {
    float4 acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = f4(0.0f);
    for (int ch = 0; ch < echunks; ++ch) {
      const int e0 = ch * kMixE, ne = min(kMixE, E - e0);
      __syncthreads();
      if (s0 == 0 || echunks > 1)
        for (int e = rg; e < ne; e += 4)
          *reinterpret_cast<float4*>(xs + e * kMixCols + col) = load4<T, kVec>(X + (e0 + e) * P, p0 + col, P);
      for (int i = threadIdx.x; i < ne * kMixRows; i += 256) {
        const int e = i / kMixRows, r = i % kMixRows;
        cf[i] = s0 + r < S ? c[(s0 + r) * cs + (e0 + e) * ce] : 0.0f;
      }
      __syncthreads();
      if (s0 + rg * 8 < S) {
#pragma unroll 4
        for (int e = 0; e < ne; ++e) {
          const float4 x = *reinterpret_cast<const float4*>(xs + e * kMixCols + col);
          const float4 a = *reinterpret_cast<const float4*>(cf + e * kMixRows + rg * 8);
          const float4 b = *reinterpret_cast<const float4*>(cf + e * kMixRows + rg * 8 + 4);
          fma4(acc[0], a.x, x); fma4(acc[1], a.y, x); fma4(acc[2], a.z, x); fma4(acc[3], a.w, x);
          fma4(acc[4], b.x, x); fma4(acc[5], b.y, x); fma4(acc[6], b.z, x); fma4(acc[7], b.w, x);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = s0 + rg * 8 + i;
      if (s < S) store4<T, kVec>(out + s * P, p0 + col, P, acc[i]);
    }
  }
}

// dc partial sums: block (split, s-tile, e-tile) adds the products of its share of the columns; a thread has
// 4 x 4 of the 64 x 64 (s, e) pairs.
constexpr int kDcCols = 64, kDcPad = kDcCols + 4;

template <typename T, bool kVec>
__global__ void __launch_bounds__(256) mix_dcoeff_kernel(const T* __restrict__ dW, const T* __restrict__ X, int S, int E,
                                                         int64_t P, int64_t share, float* __restrict__ part) {
  __shared__ float ds[64][kDcPad], xs[64][kDcPad];
  const int s0 = blockIdx.y * 64, e0 = blockIdx.z * 64;
  const int ts = threadIdx.x >> 4, te = threadIdx.x & 15;
  const int64_t pa = (int64_t)blockIdx.x * share, pb = min(P, pa + share);
  float acc[4][4] = {};
  for (int64_t p = pa; p < pb; p += kDcCols) {
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * (kDcCols / 4); i += 256) {
      const int r = i / (kDcCols / 4), q = (i % (kDcCols / 4)) * 4;
      *reinterpret_cast<float4*>(&ds[r][q]) = s0 + r < S ? load4<T, kVec>(dW + (s0 + r) * P, p + q, pb) : f4(0.0f);
      *reinterpret_cast<float4*>(&xs[r][q]) = e0 + r < E ? load4<T, kVec>(X + (e0 + r) * P, p + q, pb) : f4(0.0f);
    }
    __syncthreads();
#pragma unroll 4
    for (int q = 0; q < kDcCols; q += 4) {
      float4 a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(&ds[ts + 16 * i][q]);
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4*>(&xs[te + 16 * j][q]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += dot4(a[i], b[j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int s = s0 + ts + 16 * i, e = e0 + te + 16 * j;
      if (s < S && e < E) part[((int64_t)blockIdx.x * S + s) * E + e] = acc[i][j];
    }
}

// dc[i] = sum over the splits, in order, in fp64: one warp per entry.
__global__ void __launch_bounds__(256) mix_dcoeff_join_kernel(const float* __restrict__ part, int splits, int64_t n,
                                                              float* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  __shared__ double sm[8][32];
  const int w = threadIdx.x >> 5;
  double s = 0.0;
  if (i < n)
    for (int k = w; k < splits; k += 8) s += (double)part[k * n + i];
  sm[w][threadIdx.x & 31] = s;
  __syncthreads();
  if (w == 0 && i < n) {
    double t = sm[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < 8; ++k) t += sm[k][threadIdx.x];
    out[i] = (float)t;
  }
}

// ---- the same maps on the tensor cores ----------------------------------------------------------
// Both maps are products with one short side on each matrix: out [M, P] = A [M, K] R [K, P] with A the
// coefficients (forward: A = c, R = X; experts' gradient: A = c^T, R = dW). They are bound by the bytes of R and
// out as long as the products are not done one by one: at S = 64, E = 32 each element read takes part in 64 of them.
// The backward pass also needs dc = dW X^T, a contraction over P of the tile that is in shared memory already, so
// ONE kernel reads dW and X once and gives both gradients.
//
// A tile of R is stored [row][64 columns] (128-byte rows, 128-byte swizzle). Read with the contraction along
// the rows it is the MN-major B operand of out; read with the contraction along the columns it is the
// K-major A operand of dc. X's tile is the K-major B operand of dc.
//
// 16-bit matrices: the coefficients are three planes of the matrices' type that add up to their 24 bits (fp16: each row
// of A scaled by a power of two into fp16's range first, undone in the epilogue), so every product is
// exact. fp32 matrices: three bf16 planes on both sides and the six products of grouped.cu, in a main and
// a cross accumulator. dc leaves TMEM for fp32 registers after every tile, each addition there rounded to
// nearest, and each CTA's sums go to a slot of their own.
//
// 640 threads, one CTA per SM: warp 0 issues the MMAs; warp 4 loads 16-bit R and X by TMA, or warps 4-11 load them through
// registers (fp32, and rows of any alignment; two warpgroups take turns, so one's loads are in flight while the
// other converts); warps 12-19 are the epilogue.
constexpr int kMixTcThreads = 640;
constexpr int kMixTcMax = 128;   // rows of A, of R and of X
constexpr int kMixCtrlRegs = 48, kMixLoadRegs = 104, kMixEpiRegs = 112;   // 640 x 96 at launch = 128 x (48 + 2 x 104 + 2 x 112)

struct MixTcArgs {
  const float* c;
  int64_t cm, ck;        // strides of the coefficient of (row of A, column of A)
  const void* R;
  const void* X;         // backward only
  void* out;
  float* part;           // backward only: [gridDim.x][K][M]
  int M, K;
  int64_t P;
  int stages;
  int tma;               // 16-bit rows loaded by TMA
  int* err;
};

__device__ __forceinline__ uint64_t mix_desc_mn(uint32_t addr, uint32_t chunk) {   // MN-major, 128-byte swizzle
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)(chunk >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}

// One elected lane of a converged warp issues.
__device__ __forceinline__ void mix_mma(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

__device__ __forceinline__ void mix_commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void mix_tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// x as three numbers of type H that add up to it: H(x), H(x - p0), H(x - p0 - p1). Not finite: p0 alone.
template <typename H>
__device__ __forceinline__ void three_planes(float x, H (&p)[3]) {
  H h = from_f32<H>(x);
  if constexpr (__is_same(H, __nv_bfloat16))
    if (__hisinf(h) && fabsf(x) <= 3.402823466e38f) h = __float2bfloat16_rz(x);
  const float r1 = fabsf(x) <= 3.402823466e38f ? x - to_f32(h) : 0.0f;
  const H m = from_f32<H>(r1);
  p[0] = h;
  p[1] = m;
  p[2] = from_f32<H>(r1 - to_f32(m));
}

__host__ __device__ inline int ceil16(int n) { return (n + 15) / 16 * 16; }

template <typename T>
struct MixTc {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kBN = kF32 ? 64 : 128;          // columns per tile
  static constexpr int kPlanesR = kF32 ? 3 : 1;
  static constexpr int kChunks = kBN / 64;
  static constexpr int kUnit = kF32 ? 4 : 8;           // values per 16 bytes of global memory
  static constexpr int kD1 = kF32 ? 2 * kBN : kBN;     // TMEM columns of one out buffer (main + cross)
  static int stage_bytes(int K, int M, bool dc) { return kPlanesR * kChunks * 128 * (ceil16(K) + (dc ? ceil16(M) : 0)); }
  static int coeff_bytes(int K, int M) { return 3 * ((K + 63) / 64) * ceil16(M) * 128; }
  static constexpr int kStaging = 8 * 4096;
  static constexpr int kFixed = kStaging + 1024 /*barriers, row scales*/ + 1024 /*alignment*/;
};

template <typename T, bool kDc>
__global__ void __launch_bounds__(kMixTcThreads, 1) mix_tc_kernel(const __grid_constant__ CUtensorMap tmR,
                                                                       const __grid_constant__ CUtensorMap tmX,
                                                                       const __grid_constant__ MixTcArgs p) {
  using L = MixTc<T>;
  constexpr bool kF32 = L::kF32;
  using H = std::conditional_t<kF32, __nv_bfloat16, T>;   // operand type
  constexpr bool kFp16 = __is_same(T, __half);
  constexpr int kBN = L::kBN, kPR = L::kPlanesR;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int m_first = blockIdx.y * kMixTcMax;             // forward: slices of 128 rows of A
  const int M = min(p.M - m_first, kMixTcMax), K = p.K;
  const int rm = ceil16(M), rk = ceil16(K), kc = (K + 63) / 64;
  const int tile_r = kPR * L::kChunks * rk * 128, tile_x = kDc ? kPR * L::kChunks * rm * 128 : 0;
  const int stage_bytes = tile_r + tile_x;
  // [stages][A planes][staging][barriers]: the MMA reads 128 rows of a tile that holds fewer; what lies
  // behind is read too (rows of the result that nobody reads), and stays inside this block
  uint8_t* smem_a = smem + p.stages * stage_bytes;
  uint8_t* smem_c = smem_a + 3 * kc * rm * 128;
  uint64_t* bar_full = reinterpret_cast<uint64_t*>(smem_c + L::kStaging);
  uint64_t* bar_empty = bar_full + 8;
  uint64_t* bar_acc_full = bar_empty + 8;
  uint64_t* bar_acc_empty = bar_acc_full + 2;
  uint64_t* bar_dc_empty = bar_acc_empty + 2;
  uint64_t* bar_done = bar_dc_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* row_scale = reinterpret_cast<float*>(tmem_slot + 2);   // [128]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 8; ++s) {
      mbar_init(&bar_full[s], p.tma ? 1 : 128);
      mbar_init(&bar_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bar_acc_full[b], 1);
      mbar_init(&bar_acc_empty[b], 256);
    }
    mbar_init(bar_dc_empty, 256);
    mbar_init(bar_done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // coefficient planes: one warp per row of A
  for (int m = warp; m < rm; m += kMixTcThreads / 32) {
    float v[4], inv = 1.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = lane + 32 * j;
      v[j] = (m < M && k < K) ? p.c[(int64_t)(m_first + m) * p.cm + (int64_t)k * p.ck] : 0.0f;
    }
    if constexpr (kFp16) {
      // largest finite magnitude of the row to [2^14, 2^15)
      uint32_t mx = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t b = __float_as_uint(v[j]) & 0x7fffffffu;
        if (b < 0x7f800000u) mx = max(mx, b);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(kFull, mx, o));
      int e = (int)(mx >> 23) - 127 - 14;
      if (e < -126) e = -126;
      inv = __uint_as_float((uint32_t)(127 - e) << 23);
      if (lane == 0) row_scale[m] = __uint_as_float((uint32_t)(127 + e) << 23);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = lane + 32 * j;
      if (k < kc * 64) {
        H pl[3];
        three_planes<H>(v[j] * inv, pl);
#pragma unroll
        for (int q = 0; q < 3; ++q)
          *reinterpret_cast<H*>(smem_a + (q * kc + k / 64) * rm * 128 + m * 128 + ((((k & 63) >> 3) ^ (m & 7)) << 4) +
                                (k & 7) * 2) = pl[q];
      }
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const int64_t tiles = (p.P + kBN - 1) / kBN;
  const uint32_t dc_tmem = tmem + 2 * L::kD1;   // dc: main at +0, cross at +128

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMixCtrlRegs));
    if (warp == 0) {
      const uint32_t fmt = kFp16 ? 0u : 1u;
      const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((uint32_t)(kBN >> 3) << 17) | (8u << 24);
      const uint32_t idesc_dc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(rm >> 3) << 17) | (8u << 24);
      // the whole warp runs the loop and one lane issues; descriptors are made once (first stage, first plane, first step)
      // and moved by their address fields, in units of 16 bytes: up to 72 MMAs of 32 cycles make a tile
      const uint32_t a0 = smem_u32(smem_a), r0 = smem_u32(smem);
      const uint64_t da0 = smem_desc_sw128(a0), db0 = mix_desc_mn(r0, kPR * rk * 128);
      const uint64_t ra0 = smem_desc_sw128(r0), xb0 = smem_desc_sw128(r0 + tile_r);
      const uint32_t plane_a = kc * rm * 8, plane_r = rk * 8, plane_x = rm * 8;
      const uint32_t tm = __shfl_sync(kFull, tmem, 0);
      const int ksteps = rk / 16;
      int it = 0, s = 0, phase = 0;
      bool ok = true;
      for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++it) {
        const int buf = it & 1;
        ok = it < 2 || mbar_wait(&bar_acc_empty[buf], ((it >> 1) - 1) & 1, abort_flag, p.err, kErrWaitAccEmpty);
        ok = ok && mbar_wait(&bar_full[s], phase, abort_flag, p.err, kErrWaitFull);
        ok = __all_sync(kFull, ok);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t at = (uint32_t)(s * (stage_bytes / 16)), d1 = tm + buf * L::kD1;
        for (int kk = 0; kk < ksteps; ++kk) {
          const uint32_t acc = kk ? 1u : 0u;
          const uint64_t da = da0 + (uint32_t)((kk >> 2) * rm * 8 + (kk & 3) * 2), db = db0 + at + kk * 128;
          mix_mma(d1, da, db, idesc, acc);
          if constexpr (kF32) {
            const uint32_t cross = d1 + kBN;
            mix_mma(cross, da, db + plane_r, idesc, acc);
            mix_mma(cross, da + plane_a, db, idesc, 1u);
            mix_mma(cross, da + plane_a, db + plane_r, idesc, 1u);
            mix_mma(cross, da, db + 2 * plane_r, idesc, 1u);
            mix_mma(cross, da + 2 * plane_a, db, idesc, 1u);
          } else {
            mix_mma(d1, da + plane_a, db, idesc, 1u);
            mix_mma(d1, da + 2 * plane_a, db, idesc, 1u);
          }
        }
        if constexpr (kDc) {
          ok = it < 1 || mbar_wait(bar_dc_empty, (it - 1) & 1, abort_flag, p.err, kErrWaitAccEmpty);
          ok = __all_sync(kFull, ok);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t dc = tm + 2 * L::kD1;
#pragma unroll
          for (int kk = 0; kk < kBN / 16; ++kk) {
            const uint32_t acc = kk ? 1u : 0u;
            const uint64_t da = ra0 + at + (uint32_t)((kk >> 2) * kPR * rk * 8 + (kk & 3) * 2);
            const uint64_t db = xb0 + at + (uint32_t)((kk >> 2) * kPR * rm * 8 + (kk & 3) * 2);
            mix_mma(dc, da, db, idesc_dc, acc);
            if constexpr (kF32) {
              const uint32_t cross = dc + 128;
              mix_mma(cross, da, db + plane_x, idesc_dc, acc);
              mix_mma(cross, da + plane_r, db, idesc_dc, 1u);
              mix_mma(cross, da + plane_r, db + plane_x, idesc_dc, 1u);
              mix_mma(cross, da, db + 2 * plane_x, idesc_dc, 1u);
              mix_mma(cross, da + 2 * plane_r, db, idesc_dc, 1u);
            }
          }
        }
        mix_commit(&bar_empty[s]);
        mix_commit(&bar_acc_full[buf]);
        if (++s == p.stages) {
          s = 0;
          phase ^= 1;
        }
      }
      __syncwarp();
      mix_commit(bar_done);
      for (uint32_t i = 0; i < kWaitLimit && !mbar_try(bar_done, 0); ++i) {
      }
      __syncwarp();
    }
  } else if (warp < 12) {
    // ---------------- loads: this warpgroup's tiles are every second one of the CTA's
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMixLoadRegs));
    const int wg = (warp - 4) >> 2, t = threadIdx.x - 128 - wg * 128;
    if (!kF32 && p.tma) {
      // 16-bit matrices whose rows TMA can address: one warp, [64 columns x all rows] per load
      if (warp == 4) {
        int it = 0;
        bool ok = true;
        for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++it) {
          const int s = it % p.stages;
          ok = it < p.stages || mbar_wait(&bar_empty[s], ((it / p.stages) - 1) & 1, abort_flag, p.err, kErrWaitEmpty);
          ok = __all_sync(kFull, ok);
          if (!ok) break;
          if (lane == 0) {
            mbar_expect_tx(&bar_full[s], stage_bytes);
            uint8_t* st = smem + s * stage_bytes;
#pragma unroll
            for (int c = 0; c < L::kChunks; ++c) {
              tma_load_2d(st + c * rk * 128, &tmR, (int)(tile * kBN) + c * 64, 0, &bar_full[s]);
              if (kDc) tma_load_2d(st + tile_r + c * rm * 128, &tmX, (int)(tile * kBN) + c * 64, 0, &bar_full[s]);
            }
          }
          __syncwarp();
        }
        if (*abort_flag && lane == 0) {
          for (int j = it - 1; j >= 0 && j >= it - p.stages; --j) {
            for (uint32_t i = 0; i < kWaitLimit && !mbar_try(&bar_full[j % p.stages], (j / p.stages) & 1); ++i) {
            }
          }
        }
        __syncwarp();
      }
    } else {
    const T* R = static_cast<const T*>(p.R);
    const T* X = static_cast<const T*>(p.X);
    const bool vec = p.P % L::kUnit == 0;
    const int units = (rk + (kDc ? rm : 0)) / 8;     // 16-byte units of this thread: 16 per row, 8 rows per round
    const int u = t & 15, row0 = t >> 4;
    constexpr int kBatch = 8;
    int it = wg;
    bool ok = true;
    for (int64_t tile = blockIdx.x + (int64_t)wg * gridDim.x; tile < tiles && ok; tile += 2 * (int64_t)gridDim.x, it += 2) {
      const int s = it % p.stages;
      const int64_t col = tile * kBN + u * L::kUnit;
      uint8_t* st = smem + s * stage_bytes;
      uint4 v[2][kBatch];
      auto fetch = [&](int j0, uint4 (&d)[kBatch]) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const int row = row0 + (j0 + b) * 8;
          d[b] = make_uint4(0u, 0u, 0u, 0u);
          if (j0 + b >= units) continue;
          const bool is_x = kDc && row >= rk;
          const int r = is_x ? row - rk : row;
          if (r >= (is_x ? M : K)) continue;
          const T* src = (is_x ? X : R) + (int64_t)r * p.P + col;
          if (vec) {
            if (col < p.P) d[b] = __ldcs(reinterpret_cast<const uint4*>(src));
          } else {
            T h[L::kUnit];
#pragma unroll
            for (int i = 0; i < L::kUnit; ++i) h[i] = col + i < p.P ? src[i] : from_f32<T>(0.0f);
            memcpy(&d[b], h, 16);
          }
        }
      };
      fetch(0, v[0]);
      if (it >= p.stages) ok = mbar_wait(&bar_empty[s], ((it / p.stages) - 1) & 1, abort_flag, p.err, kErrWaitEmpty);
      if (!ok) break;
#pragma unroll 1
      for (int j0 = 0; j0 < units; j0 += 2 * kBatch) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int j = j0 + half * kBatch;
          if (j < units) {
            if (j + kBatch < units) fetch(j + kBatch, v[half ^ 1]);
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
              const int row = row0 + (j + b) * 8;
              if (j + b >= units) continue;
              const bool is_x = kDc && row >= rk;
              const int r = is_x ? row - rk : row, rows = is_x ? rm : rk;
              uint8_t* base = st + (is_x ? tile_r : 0) + r * 128;
              if constexpr (kF32) {
                const float f[4] = {__uint_as_float(v[half][b].x), __uint_as_float(v[half][b].y),
                                    __uint_as_float(v[half][b].z), __uint_as_float(v[half][b].w)};
                H pl[4][3];
#pragma unroll
                for (int i = 0; i < 4; ++i) three_planes<H>(f[i], pl[i]);
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                  const H h[4] = {pl[0][q], pl[1][q], pl[2][q], pl[3][q]};
                  uint2 w;
                  memcpy(&w, h, 8);
                  *reinterpret_cast<uint2*>(base + q * rows * 128 + (((u >> 1) ^ (r & 7)) << 4) + (u & 1) * 8) = w;
                }
              } else {
                *reinterpret_cast<uint4*>(base + (u >> 3) * rows * 128 + (((u & 7) ^ (r & 7)) << 4)) = v[half][b];
              }
            }
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&bar_full[s]);
    }
    }
  } else {
    // ---------------- epilogue: TMEM lane quadrant q, half of the columns
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMixEpiRegs));
    const int q = warp & 3, half = (warp - 12) >> 2;
    uint8_t* stage = smem_c + (warp - 12) * 4096;
    T* out = static_cast<T*>(p.out);
    const bool vec = p.P % L::kUnit == 0;
    constexpr int kHalfCols = kBN / 2;                   // 32 fp32 or 64 16-bit values: 128 bytes per row
    const int dc_half = (rm + 63) / 64 * 32;             // dc columns of this warp: [half * dc_half, + dc_half), at most 64
    float acc[kDc ? 64 : 1];
#pragma unroll
    for (int i = 0; i < (kDc ? 64 : 1); ++i) acc[i] = 0.0f;
    const float scale = kFp16 && q * 32 + lane < M ? row_scale[q * 32 + lane] : 1.0f;
    int it = 0;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++it) {
      const int buf = it & 1;
      bool ok = mbar_wait(&bar_acc_full[buf], (it >> 1) & 1, abort_flag, p.err, kErrWaitAcc);
      ok = __all_sync(kFull, ok && !*abort_flag);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t lanes = (uint32_t)(q * 32) << 16;
      if constexpr (kDc) {
        if (q * 32 < K) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (c * 32 < dc_half && half * dc_half + c * 32 < M) {
              uint32_t r[32];
              mix_tmem_ld32(dc_tmem + half * dc_half + c * 32 + lanes, r);
#pragma unroll
              for (int i = 0; i < 32; ++i) acc[c * 32 + i] += __uint_as_float(r[i]);
              if constexpr (kF32) {
                mix_tmem_ld32(dc_tmem + 128 + half * dc_half + c * 32 + lanes, r);
#pragma unroll
                for (int i = 0; i < 32; ++i) acc[c * 32 + i] += __uint_as_float(r[i]);
              }
            }
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive(bar_dc_empty);
      }
      if (q * 32 < M) {
        const uint32_t d1 = tmem + buf * L::kD1 + half * kHalfCols + lanes;
        const int rows = min(32, M - q * 32);
        __syncwarp();
#pragma unroll
        for (int c = 0; c < kHalfCols / 32; ++c) {
          uint32_t r[32];
          mix_tmem_ld32(d1 + c * 32, r);
          if constexpr (kF32) {
            uint32_t x[32];
            mix_tmem_ld32(d1 + kBN + c * 32, x);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<float4*>(stage + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                  make_float4(__uint_as_float(r[4 * j]) + __uint_as_float(x[4 * j]),
                              __uint_as_float(r[4 * j + 1]) + __uint_as_float(x[4 * j + 1]),
                              __uint_as_float(r[4 * j + 2]) + __uint_as_float(x[4 * j + 2]),
                              __uint_as_float(r[4 * j + 3]) + __uint_as_float(x[4 * j + 3]));
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              T h[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) h[i] = from_f32<T>(__uint_as_float(r[8 * j + i]) * scale);
              uint4 w;
              memcpy(&w, h, 16);
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((c * 4 + j) ^ (lane & 7)) << 4)) = w;
            }
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive(&bar_acc_empty[buf]);
        __syncwarp();
        const int64_t c0 = tile * kBN + half * kHalfCols;
        T* o = out + (int64_t)(m_first + q * 32) * p.P + c0;
        if (vec) {
          const int rr = lane >> 3, j = lane & 7;
          if (c0 + j * L::kUnit < p.P) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = i * 4 + rr;
              if (r < rows)
                __stcs(reinterpret_cast<uint4*>(o + r * p.P + j * L::kUnit),
                       *reinterpret_cast<const uint4*>(stage + r * 128 + ((j ^ (r & 7)) << 4)));
            }
          }
        } else {
          for (int r = 0; r < rows; ++r)
#pragma unroll
            for (int c = lane; c < kHalfCols; c += 32)
              if (c0 + c < p.P)
                o[r * p.P + c] = *reinterpret_cast<const T*>(stage + r * 128 + (((c / L::kUnit) ^ (r & 7)) << 4) +
                                                             (c % L::kUnit) * sizeof(T));
        }
      } else {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive(&bar_acc_empty[buf]);
      }
    }
    if constexpr (kDc) {
      const int s = q * 32 + lane;   // dc row; its columns are the experts (rows of X)
      if (s < K) {
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          const int e = half * dc_half + i;
          if (i < dc_half && e < M) p.part[((int64_t)blockIdx.x * K + s) * M + e] = acc[i];
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

namespace {

template <typename T, bool kVec>
cudaError_t run_mix(const float* c, int64_t cs, int64_t ce, const void* X, int S, int E, int64_t P, void* out,
                    cudaStream_t s) {
  auto kern = mix_kernel<T, kVec>;
  static thread_local uint64_t configured = 0;  // one bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(configured >> (dev & 63) & 1)) {
    const cudaError_t st = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMixSmem);
    if (st != cudaSuccess) return st;
    configured |= uint64_t(1) << (dev & 63);
  }
  kern<<<(unsigned)((P + kMixCols - 1) / kMixCols), 256, kMixSmem, s>>>(c, cs, ce, static_cast<const T*>(X), S, E, P,
                                                                       static_cast<T*>(out));
  return cudaGetLastError();
}

// Column shares: about two blocks per SM over all (s, e) tiles, at least 512 columns each.
int64_t dcoeff_share(int S, int E, int64_t P) {
  const int64_t tiles = (int64_t)((S + 63) / 64) * ((E + 63) / 64);
  int64_t splits = (2 * 148 + tiles - 1) / tiles;
  int64_t share = (P + splits - 1) / splits;
  if (share < 512) share = 512;
  return (share + kDcCols - 1) / kDcCols * kDcCols;
}

template <typename T, bool kVec>
cudaError_t run_dcoeff(const void* dW, const void* X, int S, int E, int64_t P, float* part, float* out,
                       cudaStream_t s) {
  const int64_t share = dcoeff_share(S, E, P);
  const int splits = (int)((P + share - 1) / share);
  mix_dcoeff_kernel<T, kVec><<<dim3((unsigned)splits, (unsigned)((S + 63) / 64), (unsigned)((E + 63) / 64)), 256, 0, s>>>(
      static_cast<const T*>(dW), static_cast<const T*>(X), S, E, P, share, part);
  const cudaError_t st = cudaGetLastError();
  if (st != cudaSuccess) return st;
  const int64_t n = (int64_t)S * E;
  mix_dcoeff_join_kernel<<<(unsigned)((n + 31) / 32), 256, 0, s>>>(part, splits, n, out);
  return cudaGetLastError();
}

constexpr int kSmemLimit = 227 * 1024;

template <typename T>
int tc_stages(int K, int M, bool dc) {
  const int room = kSmemLimit - MixTc<T>::kFixed - MixTc<T>::coeff_bytes(K, M < kMixTcMax ? M : kMixTcMax);
  const int n = room / MixTc<T>::stage_bytes(K, M < kMixTcMax ? M : kMixTcMax, dc);
  return n < 4 ? n : 4;
}

int tc_grid(int64_t P, int bn) {
  const int64_t tiles = (P + bn - 1) / bn;
  return (int)(tiles < sm_count() ? tiles : sm_count());
}

// Few coefficients: the vector kernels, whose blocks start at once, and several to an SM.
bool use_tc(int S, int E) { return (int64_t)S * E >= 64; }

template <typename T, bool kDc>
cudaError_t run_tc(MixTcArgs p, cudaStream_t s) {
  auto kern = mix_tc_kernel<T, kDc>;
  static thread_local uint64_t configured = 0;  // one bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(configured >> (dev & 63) & 1)) {
    const cudaError_t st = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
    if (st != cudaSuccess) return st;
    configured |= uint64_t(1) << (dev & 63);
  }
  p.stages = tc_stages<T>(p.K, p.M, kDc);
  const int m = p.M < kMixTcMax ? p.M : kMixTcMax;
  const int smem = MixTc<T>::kFixed + MixTc<T>::coeff_bytes(p.K, m) + p.stages * MixTc<T>::stage_bytes(p.K, m, kDc);
  CUtensorMap mr{}, mx{};
  p.tma = 0;
  if constexpr (sizeof(T) == 2) {
    const CUtensorMapDataType dt =
        std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    p.tma = p.P % 8 == 0 && p.P < ((int64_t)1 << 31) - 256 &&
            make_map_t(&mr, dt, p.R, p.K, p.P, p.P * 2, 64, ceil16(p.K), CU_TENSOR_MAP_SWIZZLE_128B) &&
            (!kDc || make_map_t(&mx, dt, p.X, p.M, p.P, p.P * 2, 64, ceil16(m), CU_TENSOR_MAP_SWIZZLE_128B));
  }
  kern<<<dim3((unsigned)tc_grid(p.P, MixTc<T>::kBN), (unsigned)((p.M + kMixTcMax - 1) / kMixTcMax)), kMixTcThreads, smem,
         s>>>(mr, mx, p);
  return cudaGetLastError();
}

template <typename T>
bool tc_fits(int K, int M, bool dc) {
  return K <= kMixTcMax && (!dc || M <= kMixTcMax) && tc_stages<T>(K, M, dc) >= 1;
}

template <typename T>
cudaError_t any_mix(const float* c, int64_t cs, int64_t ce, const void* X, int S, int E, int64_t P, void* out, int* err,
                    cudaStream_t s) {
  if (use_tc(S, E) && tc_fits<T>(E, S, false)) {
    MixTcArgs p{};
    p.c = c; p.cm = cs; p.ck = ce; p.R = X; p.out = out; p.M = S; p.K = E; p.P = P; p.err = err;
    return run_tc<T, false>(p, s);
  }
  return P % 4 == 0 ? run_mix<T, true>(c, cs, ce, X, S, E, P, out, s) : run_mix<T, false>(c, cs, ce, X, S, E, P, out, s);
}

template <typename T>
int64_t bwd_splits(int S, int E, int64_t P) {
  if (use_tc(S, E) && tc_fits<T>(S, E, true)) return tc_grid(P, MixTc<T>::kBN);
  const int64_t share = dcoeff_share(S, E, P);
  return (P + share - 1) / share;
}

template <typename T>
cudaError_t any_bwd(const float* c, int64_t cs, int64_t ce, const void* dW, const void* X, int S, int E, int64_t P,
                    float* dc, void* dX, float* part, int* err, cudaStream_t s) {
  if (dc && dX && use_tc(S, E) && tc_fits<T>(S, E, true)) {
    MixTcArgs p{};
    p.c = c; p.cm = ce; p.ck = cs; p.R = dW; p.X = X; p.out = dX; p.part = part; p.M = E; p.K = S; p.P = P; p.err = err;
    const cudaError_t st = run_tc<T, true>(p, s);
    if (st != cudaSuccess) return st;
    const int64_t n = (int64_t)S * E;
    mix_dcoeff_join_kernel<<<(unsigned)((n + 31) / 32), 256, 0, s>>>(part, tc_grid(P, MixTc<T>::kBN), n, dc);
    return cudaGetLastError();
  }
  if (dX) {
    const cudaError_t st = any_mix<T>(c, ce, cs, dW, E, S, P, dX, err, s);
    if (st != cudaSuccess) return st;
  }
  if (dc)
    return P % 4 == 0 ? run_dcoeff<T, true>(dW, X, S, E, P, part, dc, s) : run_dcoeff<T, false>(dW, X, S, E, P, part, dc, s);
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_mix(const float* c, int64_t cs, int64_t ce, const void* X, int S, int E, int64_t P, int dtype,
                       void* out, int* err, cudaStream_t s) {
  if (dtype == kDtypeF32) return any_mix<float>(c, cs, ce, X, S, E, P, out, err, s);
  if (dtype == kDtypeBf16) return any_mix<__nv_bfloat16>(c, cs, ce, X, S, E, P, out, err, s);
  return any_mix<__half>(c, cs, ce, X, S, E, P, out, err, s);
}

int64_t mix_bwd_work_bytes(int S, int E, int64_t P, int dtype) {
  const int64_t share = dcoeff_share(S, E, P);
  int64_t n = (P + share - 1) / share;   // the coefficients' gradient alone
  const int64_t tc = dtype == kDtypeF32 ? bwd_splits<float>(S, E, P)
                     : dtype == kDtypeBf16 ? bwd_splits<__nv_bfloat16>(S, E, P) : bwd_splits<__half>(S, E, P);
  if (tc > n) n = tc;
  return n * S * E * 4;
}

cudaError_t launch_mix_bwd(const float* c, int64_t cs, int64_t ce, const void* dW, const void* X, int S, int E, int64_t P,
                           int dtype, float* dc, void* dX, float* part, int* err, cudaStream_t s) {
  if (dtype == kDtypeF32) return any_bwd<float>(c, cs, ce, dW, X, S, E, P, dc, dX, part, err, s);
  if (dtype == kDtypeBf16) return any_bwd<__nv_bfloat16>(c, cs, ce, dW, X, S, E, P, dc, dX, part, err, s);
  return any_bwd<__half>(c, cs, ce, dW, X, S, E, P, dc, dX, part, err, s);
}

}  // namespace fuma
