// Per-system weights of a mixture of linear experts and their gradients. With a system's E coefficients
// c[s, :] and the expert matrices X[e, :] (P elements each, in any shape):
//
//   W[s, p]   = sum_e c[s, e] X[e, p]
//   dX[e, p]  = sum_s c[s, e] dW[s, p]      (the same map with c transposed)
//   dc[s, e]  = sum_p dW[s, p] X[e, p]
//
// Coefficients and their gradients are fp32, the matrices fp32, bf16 or fp16; sums are fp32, and the sum over
// P is in fp32 over at most kDcFlush columns and in fp64 from there on.
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
constexpr int kDcFlush = 4096;

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

// An fp32 sum to an fp64 slot that no other thread adds to, stored or added. Conversion and access are one statement: left
// apart, the compiler carries fp64 sums through the loops before, for want of registers (mix_tc_kernel, 64 x 32 x 491,520 bf16: 49
// us, so 39; mix_dcoeff_kernel, 160 x 96: 1,416, so 1,095).
__device__ __forceinline__ void store_f64(double* at, float v) {
  asm volatile("{\n\t.reg .f64 d;\n\tcvt.f64.f32 d, %1;\n\tst.global.f64 [%0], d;\n\t}" ::"l"(at), "f"(v) : "memory");
}
__device__ __forceinline__ void add_f64(double* at, float v) {
  asm volatile("{\n\t.reg .f64 d;\n\tcvt.f64.f32 d, %1;\n\tred.global.add.f64 [%0], d;\n\t}" ::"l"(at), "f"(v) : "memory");
}

// dc partial sums [split][e][s]: block (split, s-tile, e-tile) adds the products of its share of the columns; a thread has
// 4 x 4 of the 64 x 64 (s, e) pairs.
constexpr int kDcCols = 64, kDcPad = kDcCols + 4;

template <typename T, bool kVec>
__global__ void __launch_bounds__(256) mix_dcoeff_kernel(const T* __restrict__ dW, const T* __restrict__ X, int S, int E,
                                                         int64_t P, int64_t share, double* __restrict__ part) {
  __shared__ float ds[64][kDcPad], xs[64][kDcPad];
  const int s0 = blockIdx.y * 64, e0 = blockIdx.z * 64;
  const int ts = threadIdx.x >> 4, te = threadIdx.x & 15;
  const int64_t pa = (int64_t)blockIdx.x * share, pb = min(P, pa + share);
  for (int64_t p0 = pa; p0 < pb; p0 += kDcFlush) {
  float acc[4][4] = {};
  const int64_t p1 = min(pb, p0 + kDcFlush);
  for (int64_t p = p0; p < p1; p += kDcCols) {
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
      if (s < S && e < E) {
        double* at = part + ((int64_t)blockIdx.x * E + e) * S + s;
        if (p0 == pa) store_f64(at, acc[i][j]);
        else add_f64(at, acc[i][j]);
      }
    }
  }
}

// dc[s, e] = sum over the splits [split][e][s], in a fixed order, in fp64: 8 warps for 32 entries.
__global__ void __launch_bounds__(256) mix_dcoeff_join_kernel(const double* __restrict__ part, int splits, int S, int E,
                                                              float* __restrict__ out) {
  const int64_t n = (int64_t)S * E;
  const int64_t i = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  __shared__ double sm[8][32];
  const int w = threadIdx.x >> 5;
  double s = 0.0;
  if (i < n)
    for (int k = w; k < splits; k += 8) s += part[k * n + i];
  sm[w][threadIdx.x & 31] = s;
  __syncthreads();
  if (w == 0 && i < n) {
    double t = sm[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < 8; ++k) t += sm[k][threadIdx.x];
    out[i % S * E + i / S] = (float)t;
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
// exact. fp32: two fp16 planes on both sides, hi = fp16(x / s), lo = fp16(x / s - hi), and the products lo hi, hi lo,
// hi hi: s is a power of two per row of A and per tile of R and of X (largest magnitude to [2^14, 2^15); 22 bits for values
// down to 2^-18 of the tile's largest, 2^-40 of that below). Three bf16 planes need no scale, but six products, and the
// MMAs (N = 64 takes 60 cycles) were then what the backward pass waited for: 312 us at 128 x 64 x 524,288.
// dc leaves TMEM for fp32 registers after every tile (fp32, with the tiles' scales) or every 256 columns, each addition
// there rounded to nearest, and from there, every kDcFlush columns, to fp64 sums in a slot of the CTA's own.
//
// A tile is a short piece of up to 256 rows that lie megabytes apart. Loads and stores of the threads' own ran at 1.7 TB/s on
// it (8 warps, 256 bytes per row; a read of the same bytes), TMA at 6.5, so rows that TMA can address (16-byte multiples)
// come and go by TMA.
//
// 640 threads, one CTA per SM: warp 0 issues the MMAs; warp 1 loads R and X by TMA: 16-bit values to where the MMAs read
// them, fp32 to a raw buffer, from which warps 4-11 write the planes (in a second pass: the tile's largest magnitude has to be
// known first). Rows of any other length go through the registers of warps 4-11 (16 bits:
// two warpgroups take turns). Warps 12-19 are the epilogue.
constexpr int kMixTcThreads = 640;
constexpr int kMixTcMax = 128;   // rows of A, of R and of X
// Barriers of the operand ring and of the ring of raw tiles: tile `it` of a CTA signals slot it % kMixSlots, whichever buffer
// (it % depth, depth <= kMixSlots) it lies in. Two warpgroups take turns, and a wait by parity is only good for one that has seen the barrier's phase
// before: with as many slots as buffers, a warpgroup at a ring of one buffer would meet every second phase of its barrier and
// pass at once. With an even number of slots each warpgroup waits for every phase of every slot that it ever waits for, in
// order, and a slot's next phase cannot end before it has: that is a tile kMixSlots >= depth further on, behind its own.
constexpr int kMixSlots = 4;
constexpr int kMixCtrlRegs = 48, kMixLoadRegs = 88, kMixEpiRegs = 128;   // 640 x 96 at launch = 128 x (48 + 2 x 88 + 2 x 128)

struct MixTcArgs {
  const float* c;
  int64_t cm, ck;        // strides of the coefficient of (row of A, column of A)
  const void* R;
  const void* X;         // backward only
  void* out;
  double* part;          // backward only: [gridDim.x][M][K]
  int M, K;
  int64_t P;
  int stages;            // of operand tiles
  int tma;               // rows that TMA can address: 1, in fp32 the number of raw buffers (1 to 4); else 0
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

__device__ __forceinline__ void mix_tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// x as kN numbers of type H that add up to it: H(x), H(x - p0), ... Not finite: p0 alone.
template <typename H, int kN>
__device__ __forceinline__ void split_planes(float x, H (&p)[kN]) {
  p[0] = from_f32<H>(x);
  if constexpr (__is_same(H, __nv_bfloat16))
    if (__hisinf(p[0]) && fabsf(x) <= 3.402823466e38f) p[0] = __float2bfloat16_rz(x);
  float r = fabsf(x) <= 3.402823466e38f ? x - to_f32(p[0]) : 0.0f;
#pragma unroll
  for (int i = 1; i < kN; ++i) {
    p[i] = from_f32<H>(r);
    r -= to_f32(p[i]);
  }
}

// The power of two that brings the largest magnitude (its bits) to [2^14, 2^15), and its inverse.
__device__ __forceinline__ float2 fp16_scale(uint32_t amax_bits) {
  int e = (int)(amax_bits >> 23) - 127 - 14;
  if (e < -126) e = -126;
  return make_float2(__uint_as_float((uint32_t)(127 + e) << 23), __uint_as_float((uint32_t)(127 - e) << 23));
}

// a b as two powers of two with half the exponent each: the product of two scales may leave the fp32 range where the
// result does not.
__device__ __forceinline__ float2 half_exponents(float a, float b) {
  const int e = (int)(__float_as_uint(a) >> 23) + (int)(__float_as_uint(b) >> 23) - 254, h = e >> 1;
  return make_float2(__uint_as_float((uint32_t)(h + 127) << 23), __uint_as_float((uint32_t)(e - h + 127) << 23));
}

__host__ __device__ inline int ceil16(int n) { return (n + 15) / 16 * 16; }

template <typename T>
struct MixTc {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kBN = kF32 ? 64 : 128;          // columns per tile
  static constexpr int kPlanesR = kF32 ? 2 : 1;
  static constexpr int kPlanesA = kF32 ? 2 : 3;
  static constexpr int kChunks = kBN / 64;
  static constexpr int kUnit = kF32 ? 4 : 8;           // values per 16 bytes of global memory
  static constexpr int kDcTiles = kF32 ? 1 : 256 / kBN;   // tiles per drain of dc
  static constexpr int kFlushTiles = kDcFlush / kBN;
  static_assert(kFlushTiles % kDcTiles == 0, "a flush follows a drain");
  static int stage_bytes(int K, int M, bool dc) { return kPlanesR * kChunks * 128 * (ceil16(K) + (dc ? ceil16(M) : 0)); }
  static int coeff_bytes(int K, int M) { return kPlanesA * ((K + 63) / 64) * ceil16(M) * 128; }
  static constexpr int kStaging = 8 * 4096;
  static constexpr int kFixed = kStaging + 1024 /*barriers, scales*/ + 1024 /*alignment*/;
};

template <typename T, bool kDc>
__global__ void __launch_bounds__(kMixTcThreads, 1) mix_tc_kernel(const __grid_constant__ CUtensorMap tmR,
                                                                       const __grid_constant__ CUtensorMap tmX,
                                                                       const __grid_constant__ CUtensorMap tmO,
                                                                       const __grid_constant__ MixTcArgs p) {
  using L = MixTc<T>;
  constexpr bool kF32 = L::kF32;
  using H = std::conditional_t<kF32, __half, T>;          // operand type
  constexpr bool kFp16 = __is_same(H, __half);
  constexpr int kBN = L::kBN, kPR = L::kPlanesR, kPA = L::kPlanesA;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int m_first = blockIdx.y * kMixTcMax;             // forward: slices of 128 rows of A
  const int M = min(p.M - m_first, kMixTcMax), K = p.K;
  const int rm = ceil16(M), rk = ceil16(K), kc = (K + 63) / 64;
  const int tile_r = kPR * L::kChunks * rk * 128, tile_x = kDc ? kPR * L::kChunks * rm * 128 : 0;
  const int stage_bytes = tile_r + tile_x;
  // [stages][A planes][staging][barriers]: the MMA reads 128 rows of a tile that holds fewer; what lies
  // behind is read too (rows of the result that nobody reads), and stays inside this block
  const int raw_bytes = (rk + (kDc ? rm : 0)) * kBN * 4;   // fp32: one raw buffer
  uint8_t* smem_a = smem + p.stages * stage_bytes;
  uint8_t* smem_c = smem_a + kPA * kc * rm * 128;
  uint8_t* smem_raw_tile = smem_c + L::kStaging + 1024;    // behind the barriers
  uint64_t* bar_full = reinterpret_cast<uint64_t*>(smem_c + L::kStaging);
  uint64_t* bar_empty = bar_full + kMixSlots;
  uint64_t* bar_acc_full = bar_empty + kMixSlots;
  uint64_t* bar_acc_empty = bar_acc_full + 2;
  uint64_t* bar_dc_empty = bar_acc_empty + 2;
  uint64_t* bar_dc_full = bar_dc_empty + 2;
  uint64_t* bar_raw_full = bar_dc_full + 2;
  uint64_t* bar_raw_empty = bar_raw_full + kMixSlots;
  uint64_t* bar_done = bar_raw_empty + kMixSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* row_scale = reinterpret_cast<float*>(tmem_slot + 2);   // [128]
  float2* tile_scale = reinterpret_cast<float2*>(row_scale + 128);   // fp32: [8] of R and X, by tile
  uint32_t* tile_max = reinterpret_cast<uint32_t*>(tile_scale + 8);  // fp32: [8][4]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kMixSlots; ++s) {
      mbar_init(&bar_full[s], !kF32 && p.tma ? 1 : 128);
      mbar_init(&bar_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bar_acc_full[b], 1);
      mbar_init(&bar_acc_empty[b], 256);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bar_dc_empty[b], 256);
      mbar_init(&bar_dc_full[b], 1);

    }
    for (int b = 0; b < kMixSlots; ++b) {
      mbar_init(&bar_raw_full[b], 1);
      mbar_init(&bar_raw_empty[b], 128);
    }
    mbar_init(bar_done, 1);
    for (int i = 0; i < 32; ++i) tile_max[i] = 0;
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
      const float2 sc = fp16_scale(mx);
      inv = sc.y;
      if (lane == 0) row_scale[m] = sc.x;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = lane + 32 * j;
      if (k < kc * 64) {
        H pl[kPA];
        split_planes<H, kPA>(v[j] * inv, pl);
#pragma unroll
        for (int q = 0; q < kPA; ++q)
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
  const uint32_t dc_tmem = tmem + 2 * kBN;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMixCtrlRegs));
    if (warp == 0) {
      const uint32_t fmt = kFp16 ? 0u : 1u;   // fp16 or bf16
      const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((uint32_t)(kBN >> 3) << 17) | (8u << 24);
      const uint32_t idesc_dc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(rm >> 3) << 17) | (8u << 24);
      // the whole warp runs the loop and one lane issues; descriptors are made once (first stage, first plane, first step)
      // and moved by their address fields, in units of 16 bytes: up to 40 short MMAs make a tile
      const uint32_t a0 = smem_u32(smem_a), r0 = smem_u32(smem);
      const uint64_t da0 = smem_desc_sw128(a0), db0 = mix_desc_mn(r0, kPR * rk * 128);
      const uint64_t ra0 = smem_desc_sw128(r0), xb0 = smem_desc_sw128(r0 + tile_r);
      const uint32_t plane_a = kc * rm * 8, plane_r = rk * 8, plane_x = rm * 8;
      const uint32_t tm = __shfl_sync(kFull, tmem, 0);
      const int ksteps = rk / 16;
      int it = 0, s = 0;
      bool ok = true;
      for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++it) {
        const int buf = it & 1, slot = it % kMixSlots;
        ok = it < 2 || mbar_wait(&bar_acc_empty[buf], ((it >> 1) - 1) & 1, abort_flag, p.err, kErrWaitAccEmpty);
        ok = ok && mbar_wait(&bar_full[slot], (it / kMixSlots) & 1, abort_flag, p.err, kErrWaitFull);
        ok = __all_sync(kFull, ok);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t at = (uint32_t)(s * (stage_bytes / 16)), d1 = tm + buf * kBN;
        for (int kk = 0; kk < ksteps; ++kk) {
          const uint32_t acc = kk ? 1u : 0u;
          const uint64_t da = da0 + (uint32_t)((kk >> 2) * rm * 8 + (kk & 3) * 2), db = db0 + at + kk * 128;
          if constexpr (kF32) {   // the small products first
            mix_mma(d1, da + plane_a, db, idesc, acc);
            mix_mma(d1, da, db + plane_r, idesc, 1u);
            mix_mma(d1, da, db, idesc, 1u);
          } else {
            mix_mma(d1, da, db, idesc, acc);
            mix_mma(d1, da + plane_a, db, idesc, 1u);
            mix_mma(d1, da + 2 * plane_a, db, idesc, 1u);
          }
        }
        if constexpr (kDc) {
          const int dci = it % L::kDcTiles, dcn = it / L::kDcTiles;
          if (dci == 0) {
            ok = dcn < 2 || mbar_wait(&bar_dc_empty[dcn & 1], ((dcn >> 1) - 1) & 1, abort_flag, p.err, kErrWaitAccEmpty);
            ok = __all_sync(kFull, ok);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          }
          const uint32_t dc = tm + 2 * kBN + (dcn & 1) * 128;
#pragma unroll
          for (int kk = 0; kk < kBN / 16; ++kk) {
            const uint32_t acc = kk || dci ? 1u : 0u;
            const uint64_t da = ra0 + at + (uint32_t)((kk >> 2) * kPR * rk * 8 + (kk & 3) * 2);
            const uint64_t db = xb0 + at + (uint32_t)((kk >> 2) * kPR * rm * 8 + (kk & 3) * 2);
            if constexpr (kF32) {
              mix_mma(dc, da + plane_r, db, idesc_dc, acc);
              mix_mma(dc, da, db + plane_x, idesc_dc, 1u);
              mix_mma(dc, da, db, idesc_dc, 1u);
            } else {
              mix_mma(dc, da, db, idesc_dc, acc);
            }
          }
        }
        mix_commit(&bar_empty[slot]);
        mix_commit(&bar_acc_full[buf]);
        if (kDc && (it % L::kDcTiles == L::kDcTiles - 1 || tile + gridDim.x >= tiles)) mix_commit(&bar_dc_full[it / L::kDcTiles & 1]);
        if (++s == p.stages) s = 0;
      }
      __syncwarp();
      mix_commit(bar_done);
      for (uint32_t i = 0; i < kWaitLimit && !mbar_try(bar_done, 0); ++i) {
      }
      __syncwarp();
    }
    if (warp == 1 && p.tma) {
      // ---------------- TMA loads: [64 columns x all rows] each
      uint64_t* full = kF32 ? bar_raw_full : bar_full;
      uint64_t* empty = kF32 ? bar_raw_empty : bar_empty;
      const int depth = kF32 ? p.tma : p.stages, bytes = kF32 ? raw_bytes : stage_bytes;
      uint8_t* base = kF32 ? smem_raw_tile : smem;
      const int row_bytes = kF32 ? 256 : 128;
      int it = 0;
      bool ok = true;
      for (int64_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++it) {
        const int s = it % depth, slot = it % kMixSlots, last = it - depth;   // the tile that was here before
        ok = last < 0 || mbar_wait(&empty[last % kMixSlots], (last / kMixSlots) & 1, abort_flag, p.err, kErrWaitEmpty);
        ok = __all_sync(kFull, ok);
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(&full[slot], bytes);
          uint8_t* st = base + s * bytes;
#pragma unroll
          for (int c = 0; c < L::kChunks; ++c) {
            tma_load_2d(st + c * rk * row_bytes, &tmR, (int)(tile * kBN) + c * 64, 0, &full[slot]);
            if (kDc)
              tma_load_2d(st + L::kChunks * rk * row_bytes + c * rm * row_bytes, &tmX, (int)(tile * kBN) + c * 64, 0, &full[slot]);
          }
        }
        __syncwarp();
      }
      if (*abort_flag && lane == 0) {
        for (int j = it - 1; j >= 0 && j >= it - depth; --j) {
          for (uint32_t i = 0; i < kWaitLimit && !mbar_try(&full[j % kMixSlots], (j / kMixSlots) & 1); ++i) {
          }
        }
      }
      __syncwarp();
    }
  } else if (warp < 12) {
    // ---------------- loads: this warpgroup's tiles are every second one of the CTA's
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMixLoadRegs));
    const int wg = (warp - 4) >> 2, t = threadIdx.x - 128 - wg * 128;
    const T* R = static_cast<const T*>(p.R);
    const T* X = static_cast<const T*>(p.X);
    const int u = t & 15;                            // 16 units of 16 bytes per row of a tile
    if constexpr (kF32) {
      // the warpgroups take turns; a warpgroup goes twice over its tile, 8 rows a round: its largest magnitude, then the planes
      const int row0 = t >> 4;
      const int rounds_r = rk / 8, rounds = rounds_r + (kDc ? rm / 8 : 0);
      int it = wg;
      for (int64_t tile = blockIdx.x + (int64_t)wg * gridDim.x; tile < tiles; tile += 2 * (int64_t)gridDim.x, it += 2) {
        const int s = it % p.stages, rb = p.tma ? it % p.tma : 0;
        const int64_t col = tile * kBN + u * 4;
        const uint8_t* raw = smem_raw_tile + rb * raw_bytes + row0 * 256 + u * 16;
        auto value = [&](int j) {   // this thread's 4 columns in row row0 + 8 j of the tile; X's rows follow R's
          if (p.tma) return *reinterpret_cast<const uint4*>(raw + j * 2048);
          const bool is_x = kDc && j >= rounds_r;
          const int row = row0 + (is_x ? j - rounds_r : j) * 8;
          const float* src = (is_x ? X : R) + (int64_t)row * p.P + col;
          float h[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) h[i] = row < (is_x ? M : K) && col + i < p.P ? src[i] : 0.0f;
          uint4 w;
          memcpy(&w, h, 16);
          return w;
        };
        // (no end of the loop after a failed wait: the other threads count on this one at the barriers below)
        if (p.tma) mbar_wait(&bar_raw_full[it % kMixSlots], (it / kMixSlots) & 1, abort_flag, p.err, kErrWaitFull);
        // the tile's largest magnitudes, as bits: of R's rows and of X's. `all`: with values that are not finite, which is
        // what tells that there are any; a second round then leaves them out
        uint32_t* tm = tile_max + (it & 7) * 4;
        auto largest = [&](bool all, uint32_t* out) {
          uint32_t m2[2] = {0, 0};
#pragma unroll
          for (int h = 0; h < (kDc ? 2 : 1); ++h) {
            uint32_t m = 0;
#pragma unroll 4
            for (int j = h ? rounds_r : 0; j < (h ? rounds : rounds_r); ++j) {
              const uint4 w = value(j);
              uint32_t x[4] = {w.x & 0x7fffffffu, w.y & 0x7fffffffu, w.z & 0x7fffffffu, w.w & 0x7fffffffu};
              if (!all)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = x[i] < 0x7f800000u ? x[i] : 0u;
              m = __vimax3_u32(m, x[0], __vimax3_u32(x[1], x[2], x[3]));
            }
            m2[h] = __reduce_max_sync(kFull, m);
            if (lane == 0) atomicMax(out + h, m2[h]);
          }
          asm volatile("bar.sync %0, 128;" ::"r"(1 + wg) : "memory");
          return make_uint2(out[0], kDc ? out[1] : 0u);
        };
        uint2 big = largest(true, tm);
        const bool odd = big.x >= 0x7f800000u || big.y >= 0x7f800000u;   // the same in all 128 threads
        if (odd) big = largest(false, tm + 2);
        const float2 sr = fp16_scale(big.x), sx = fp16_scale(big.y);
        if (t == 0) {
          tile_scale[it & 7] = make_float2(sr.x, sx.x);
          // four tiles on: this warpgroup's too, nobody is there before another barrier, and everybody has left it
          *reinterpret_cast<uint4*>(tile_max + ((it + 4) & 7) * 4) = make_uint4(0u, 0u, 0u, 0u);
        }
        const int last = it - p.stages;   // the tile that was in this stage before
        const bool ok = last < 0 || mbar_wait(&bar_empty[last % kMixSlots], (last / kMixSlots) & 1, abort_flag, p.err, kErrWaitEmpty);
        uint8_t* dst = smem + s * stage_bytes + row0 * 128 + ((((u >> 1) ^ row0) & 7) << 4) + (u & 1) * 8;
        if (ok) {
#pragma unroll
          for (int h = 0; h < (kDc ? 2 : 1); ++h) {
            const float inv = h ? sx.y : sr.y;
            const int plane = (h ? rm : rk) * 128;
            uint8_t* at = dst + (h ? tile_r - rounds_r * 1024 : 0);
#pragma unroll 4
            for (int j = h ? rounds_r : 0; j < (h ? rounds : rounds_r); ++j) {
              const uint4 w = value(j);
              const float f[4] = {__uint_as_float(w.x) * inv, __uint_as_float(w.y) * inv, __uint_as_float(w.z) * inv,
                                  __uint_as_float(w.w) * inv};
              const __half2 h01 = __floats2half2_rn(f[0], f[1]), h23 = __floats2half2_rn(f[2], f[3]);
              const float2 g01 = __half22float2(h01), g23 = __half22float2(h23);
              float d[4] = {f[0] - g01.x, f[1] - g01.y, f[2] - g23.x, f[3] - g23.y};
              if (odd)
#pragma unroll
                for (int i = 0; i < 4; ++i) d[i] = fabsf(f[i]) <= 65504.0f ? d[i] : 0.0f;   // not finite: hi alone
              const __half2 l01 = __floats2half2_rn(d[0], d[1]), l23 = __floats2half2_rn(d[2], d[3]);
              *reinterpret_cast<uint2*>(at + j * 1024) = make_uint2(h2_bits(h01), h2_bits(h23));
              *reinterpret_cast<uint2*>(at + j * 1024 + plane) = make_uint2(h2_bits(l01), h2_bits(l23));
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&bar_full[it % kMixSlots]);
        if (p.tma) mbar_arrive(&bar_raw_empty[it % kMixSlots]);
      }
    } else if (!p.tma) {
    const int rounds_r = rk / 8, rounds = rounds_r + (kDc ? rm / 8 : 0);   // 8 rows a round, 16 units of 16 bytes per row
    const int row0 = t >> 4;
    const int64_t step = 8 * p.P;
    constexpr int kBatch = 4;
    int it = wg;
    bool ok = true;
    for (int64_t tile = blockIdx.x + (int64_t)wg * gridDim.x; tile < tiles && ok; tile += 2 * (int64_t)gridDim.x, it += 2) {
      const int s = it % p.stages;
      const int64_t col = tile * kBN + u * L::kUnit;
      const T* src_r = R + row0 * p.P + col;
      const T* src_x = X + row0 * p.P + col - rounds_r * step;
      uint4 v[2][kBatch];
      auto fetch = [&](int j0, uint4 (&d)[kBatch]) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const int j = j0 + b;
          const bool is_x = kDc && j >= rounds_r;
          const int row = row0 + (is_x ? j - rounds_r : j) * 8;
          const T* src = (is_x ? src_x : src_r) + j * step;
          d[b] = make_uint4(0u, 0u, 0u, 0u);
          if (j < rounds && row < (is_x ? M : K)) {
            T h[L::kUnit];
#pragma unroll
            for (int i = 0; i < L::kUnit; ++i) h[i] = col + i < p.P ? src[i] : from_f32<T>(0.0f);
            memcpy(&d[b], h, 16);
          }
        }
      };
      fetch(0, v[0]);
      const int last = it - p.stages;   // the tile that was in this stage before
      if (last >= 0) ok = mbar_wait(&bar_empty[last % kMixSlots], (last / kMixSlots) & 1, abort_flag, p.err, kErrWaitEmpty);
      if (!ok) break;
      // this thread's 16 bytes in row row0 of a tile; rows 8 further on are 1024 bytes on and
      // have the same swizzle
      uint8_t* dst = smem + s * stage_bytes + row0 * 128 + (((u ^ row0) & 7) << 4);
#pragma unroll 1
      for (int j0 = 0; j0 < rounds; j0 += 2 * kBatch) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int j = j0 + half * kBatch;
          if (j < rounds) {
            if (j + kBatch < rounds) fetch(j + kBatch, v[half ^ 1]);
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
              if (j + b >= rounds) break;
              const bool is_x = kDc && j + b >= rounds_r;
              const int plane = (is_x ? rm : rk) * 128;
              uint8_t* at = dst + (is_x ? tile_r + (j + b - rounds_r) * 1024 : (j + b) * 1024);
              *reinterpret_cast<uint4*>(at + (u >> 3) * plane) = v[half][b];
            }
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&bar_full[it % kMixSlots]);
    }
    }
  } else {
    // ---------------- epilogue: TMEM lane quadrant q, half of the columns
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMixEpiRegs));
    const int q = warp & 3, half = (warp - 12) >> 2;
    uint8_t* stage = smem_c + (warp - 12) * 4096;
    T* out = static_cast<T*>(p.out);
    constexpr int kHalfCols = kBN / 2;                   // 32 fp32 or 64 16-bit values: 128 bytes per row
    const int dc_half = (rm + 63) / 64 * 32;             // dc columns of this warp: [half * dc_half, + dc_half), at most 64
    float acc[kDc ? 64 : 1];
#pragma unroll
    for (int i = 0; i < (kDc ? 64 : 1); ++i) acc[i] = 0.0f;
    const float scale = kFp16 && q * 32 + lane < M ? row_scale[q * 32 + lane] : 1.0f;
    // the register sums to the CTA's fp64 slot, which this thread alone adds to: dc row s = R's row, one per lane
    auto add_dc = [&](bool first) {
      const int s = q * 32 + lane, e0 = half * dc_half;
      double* part = p.part + ((int64_t)blockIdx.x * M + e0) * K + s;
      int n = s < K ? min(dc_half, M - e0) : 0;
      asm volatile("" : "+r"(n));   // opaque, or 64 predicates are made before the loop over the tiles and kept
      // one loop or the other: a choice for each entry cost 4 us of 39
      if (first) {
#pragma unroll
        for (int i = 0; i < (kDc ? 64 : 1); ++i, part += K)
          if (i < n) store_f64(part, acc[i]);
      } else {
#pragma unroll
        for (int i = 0; i < (kDc ? 64 : 1); ++i, part += K)
          if (i < n) add_f64(part, acc[i]);
      }
#pragma unroll
      for (int i = 0; i < (kDc ? 64 : 1); ++i) acc[i] = 0.0f;
    };
    int it = 0;
    bool ok = true;
    int64_t tile = blockIdx.x;
    do {   // backward: runs of kDcFlush columns
    const int it_end = it + L::kFlushTiles;
    for (; tile < tiles && (!kDc || it < it_end); tile += gridDim.x, ++it) {
      const int buf = it & 1;
      ok = mbar_wait(&bar_acc_full[buf], (it >> 1) & 1, abort_flag, p.err, kErrWaitAcc);
      ok = __all_sync(kFull, ok && !*abort_flag);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t lanes = (uint32_t)(q * 32) << 16;
      const float2 ts = kF32 ? tile_scale[it & 7] : make_float2(1.0f, 1.0f);   // the ring is longer than anyone is ahead
      auto drain_dc = [&]() {   // TMEM's sum of the last tiles to registers, rounded to nearest
        const int dcn = it / L::kDcTiles;
        bool full = mbar_wait(&bar_dc_full[dcn & 1], (dcn >> 1) & 1, abort_flag, p.err, kErrWaitAcc);
        full = __all_sync(kFull, full && !*abort_flag);
        if (!full) return false;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const float2 sc = half_exponents(ts.x, ts.y);
        if (q * 32 < K) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (c * 16 < dc_half && half * dc_half + c * 16 < M) {
              uint32_t r[16];
              mix_tmem_ld16(dc_tmem + (dcn & 1) * 128 + half * dc_half + c * 16 + lanes, r);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                if constexpr (kF32) acc[c * 16 + i] = fmaf(__uint_as_float(r[i]) * sc.x, sc.y, acc[c * 16 + i]);
                else acc[c * 16 + i] += __uint_as_float(r[i]);
              }
            }
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive(&bar_dc_empty[dcn & 1]);
        return true;
      };
      if (q * 32 < M) {
        const uint32_t d1 = tmem + buf * kBN + half * kHalfCols + lanes;
        const int rows = min(32, M - q * 32);
        const float2 so = kF32 ? half_exponents(scale, ts.x) : make_float2(scale, 1.0f);
        if (p.tma && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int c = 0; c < kHalfCols / 32; ++c) {
          if constexpr (kF32) {
            uint32_t r[32];
            mix_tmem_ld32(d1, r);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float o[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) o[i] = __uint_as_float(r[4 * j + i]) * so.x * so.y;
              *reinterpret_cast<float4*>(stage + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_float4(o[0], o[1], o[2], o[3]);
            }
          } else {
            uint32_t r[32];
            mix_tmem_ld32(d1 + c * 32, r);
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
        if (p.tma) {   // rows behind the last and columns behind P are clipped
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                             reinterpret_cast<uint64_t>(&tmO)),
                         "r"((int)c0), "r"(m_first + q * 32), "r"(smem_u32(stage))
                         : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
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
      if constexpr (kDc) {
        if (it % L::kDcTiles == L::kDcTiles - 1 || tile + gridDim.x >= tiles) {
          ok = drain_dc();
          if (!ok) break;
        }
      }
    }
    if constexpr (kDc) add_dc(it <= L::kFlushTiles);
    } while (kDc && ok && tile < tiles);
    if (p.tma && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // the staging area outlives its reads
    __syncwarp();
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
  int64_t splits = (2 * sm_count() + tiles - 1) / tiles;
  int64_t share = (P + splits - 1) / splits;
  if (share < 512) share = 512;
  return (share + kDcCols - 1) / kDcCols * kDcCols;
}

template <typename T, bool kVec>
cudaError_t run_dcoeff(const void* dW, const void* X, int S, int E, int64_t P, double* part, float* out,
                       cudaStream_t s) {
  const int64_t share = dcoeff_share(S, E, P);
  const int splits = (int)((P + share - 1) / share);
  mix_dcoeff_kernel<T, kVec><<<dim3((unsigned)splits, (unsigned)((S + 63) / 64), (unsigned)((E + 63) / 64)), 256, 0, s>>>(
      static_cast<const T*>(dW), static_cast<const T*>(X), S, E, P, share, part);
  const cudaError_t st = cudaGetLastError();
  if (st != cudaSuccess) return st;
  mix_dcoeff_join_kernel<<<(unsigned)(((int64_t)S * E + 31) / 32), 256, 0, s>>>(part, splits, S, E, out);
  return cudaGetLastError();
}

constexpr int kSmemLimit = 227 * 1024;

// Operand stages that fit beside the coefficients, the staging area and, in fp32, `raw` raw tiles.
template <typename T>
int tc_stages(int K, int M, bool dc, int raw) {
  const int m = M < kMixTcMax ? M : kMixTcMax;
  const int tile = MixTc<T>::stage_bytes(K, m, dc);
  const int raw_bytes = sizeof(T) == 4 ? raw * (tile / MixTc<T>::kPlanesR / 2 * 4) : 0;
  const int n = (kSmemLimit - MixTc<T>::kFixed - MixTc<T>::coeff_bytes(K, m) - raw_bytes) / tile;
  return n < kMixSlots ? n : kMixSlots;
}

int tc_grid(int64_t P, int bn) {
  const int64_t tiles = (P + bn - 1) / bn;
  return (int)(tiles < sm_count() ? tiles : sm_count());
}

// Forward: few coefficients go to the vector kernel, whose blocks start at once, and several to an SM; its time grows
// with S E, that of the tensor-core kernel hardly. Rows that TMA cannot read (not a multiple of 16 bytes apart) cost the
// latter more. us, vector and tensor cores, for matrices of 491,520 values (odd: 102,307):
//   bf16  S E = 128  19.8, 17.6 (of 16,384 values 4.3, 5.1); 512  36.7, 19.2;  odd 1024  15.0, 21.7; 2048  25.1, 23.0
//   fp32  S E = 512  38.2, 53.6; 1024  54.8, 54.6; 2048  90.6, 56.7;           odd 2048  23.5, 34.9
// Both gradients at once always go to the tensor cores, which read the matrices once: bf16 S E = 8 30 + 3,
// vector 13 + 127 + 5; fp32 89 + 4, vector 13 + 125 + 5. (dc alone takes the vector kernel at every size: the one-pass kernel
// has no form without dX.)
template <typename T>
bool use_tc(int S, int E, int64_t P) {
  const bool aligned = P * sizeof(T) % 16 == 0;
  return (int64_t)S * E >= (sizeof(T) == 2 ? (aligned ? 256 : 2048) : (aligned ? 1024 : 4096));
}

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
  const int m = p.M < kMixTcMax ? p.M : kMixTcMax;
  constexpr bool kF32 = sizeof(T) == 4;
  CUtensorMap mr{}, mx{}, mo{};
  const CUtensorMapDataType dt = kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                             : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapSwizzle sw = kF32 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B;
  const int64_t pitch = p.P * (int64_t)sizeof(T);
  // fp32: two raw buffers (one per splitting warpgroup) come first, then two operand stages, then more raw buffers
  const int raw = !kF32 ? 1 : tc_stages<T>(p.K, p.M, kDc, 4) >= 2 ? 4 : tc_stages<T>(p.K, p.M, kDc, 2) >= 1 ? 2 : 1;
  const bool tma = pitch % 16 == 0 && p.P < ((int64_t)1 << 31) - 256 && tc_stages<T>(p.K, p.M, kDc, raw) >= 1 &&
          make_map_t(&mr, dt, p.R, p.K, p.P, pitch, 64, ceil16(p.K), sw) &&
          (!kDc || make_map_t(&mx, dt, p.X, p.M, p.P, pitch, 64, ceil16(m), sw)) &&
          make_map_t(&mo, dt, p.out, p.M, p.P, pitch, 128 / sizeof(T), 32, CU_TENSOR_MAP_SWIZZLE_128B);
  p.tma = tma ? raw : 0;
  p.stages = tc_stages<T>(p.K, p.M, kDc, p.tma);
  const int tile = MixTc<T>::stage_bytes(p.K, m, kDc);
  const int smem = MixTc<T>::kFixed + MixTc<T>::coeff_bytes(p.K, m) + p.stages * tile +
                   (kF32 ? p.tma * (tile / MixTc<T>::kPlanesR / 2 * 4) : 0);
  kern<<<dim3((unsigned)tc_grid(p.P, MixTc<T>::kBN), (unsigned)((p.M + kMixTcMax - 1) / kMixTcMax)), kMixTcThreads, smem,
         s>>>(mr, mx, mo, p);
  return cudaGetLastError();
}

template <typename T>
bool tc_fits(int K, int M, bool dc) {
  return K <= kMixTcMax && (!dc || M <= kMixTcMax) && tc_stages<T>(K, M, dc, 0) >= 1;
}

template <typename T>
cudaError_t any_mix(const float* c, int64_t cs, int64_t ce, const void* X, int S, int E, int64_t P, void* out, int* err,
                    cudaStream_t s) {
  if (use_tc<T>(S, E, P) && tc_fits<T>(E, S, false)) {
    MixTcArgs p{};
    p.c = c; p.cm = cs; p.ck = ce; p.R = X; p.out = out; p.M = S; p.K = E; p.P = P; p.err = err;
    return run_tc<T, false>(p, s);
  }
  return P % 4 == 0 ? run_mix<T, true>(c, cs, ce, X, S, E, P, out, s) : run_mix<T, false>(c, cs, ce, X, S, E, P, out, s);
}

template <typename T>
int64_t bwd_splits(int S, int E, int64_t P) {
  if (tc_fits<T>(S, E, true)) return tc_grid(P, MixTc<T>::kBN);
  const int64_t share = dcoeff_share(S, E, P);
  return (P + share - 1) / share;
}

template <typename T>
cudaError_t any_bwd(const float* c, int64_t cs, int64_t ce, const void* dW, const void* X, int S, int E, int64_t P,
                    float* dc, void* dX, double* part, int* err, cudaStream_t s) {
  if (dc && dX && tc_fits<T>(S, E, true)) {
    MixTcArgs p{};
    p.c = c; p.cm = ce; p.ck = cs; p.R = dW; p.X = X; p.out = dX; p.part = part; p.M = E; p.K = S; p.P = P; p.err = err;
    const cudaError_t st = run_tc<T, true>(p, s);
    if (st != cudaSuccess) return st;
    mix_dcoeff_join_kernel<<<(unsigned)(((int64_t)S * E + 31) / 32), 256, 0, s>>>(part, tc_grid(P, MixTc<T>::kBN), S, E, dc);
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

int mix_bwd_launches(int S, int E, int dtype, bool dc, bool dX) {
  const bool tc = dtype == kDtypeF32 ? tc_fits<float>(S, E, true)
                  : dtype == kDtypeBf16 ? tc_fits<__nv_bfloat16>(S, E, true) : tc_fits<__half>(S, E, true);
  return dc && dX && tc ? 2 : (dX ? 1 : 0) + (dc ? 2 : 0);   // any_bwd
}

int64_t mix_bwd_work_bytes(int S, int E, int64_t P, int dtype) {
  const int64_t share = dcoeff_share(S, E, P);
  int64_t n = (P + share - 1) / share;   // the coefficients' gradient alone
  const int64_t tc = dtype == kDtypeF32 ? bwd_splits<float>(S, E, P)
                     : dtype == kDtypeBf16 ? bwd_splits<__nv_bfloat16>(S, E, P) : bwd_splits<__half>(S, E, P);
  if (tc > n) n = tc;
  return n * S * E * 8;
}

cudaError_t launch_mix_bwd(const float* c, int64_t cs, int64_t ce, const void* dW, const void* X, int S, int E, int64_t P,
                           int dtype, float* dc, void* dX, double* part, int* err, cudaStream_t s) {
  if (dtype == kDtypeF32) return any_bwd<float>(c, cs, ce, dW, X, S, E, P, dc, dX, part, err, s);
  if (dtype == kDtypeBf16) return any_bwd<__nv_bfloat16>(c, cs, ce, dW, X, S, E, P, dc, dX, part, err, s);
  return any_bwd<__half>(c, cs, ce, dW, X, S, E, P, dc, dX, part, err, s);
}

}  // namespace fuma
