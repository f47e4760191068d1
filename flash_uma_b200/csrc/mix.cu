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

#include "common.cuh"
#include "grouped.cuh"
#include "kernels.h"

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

}  // namespace

cudaError_t launch_mix(const float* c, int64_t cs, int64_t ce, const void* X, int S, int E, int64_t P, int dtype,
                       void* out, cudaStream_t s) {
  const bool vec = P % 4 == 0;
  if (dtype == kDtypeF32)
    return vec ? run_mix<float, true>(c, cs, ce, X, S, E, P, out, s) : run_mix<float, false>(c, cs, ce, X, S, E, P, out, s);
  if (dtype == kDtypeBf16)
    return vec ? run_mix<__nv_bfloat16, true>(c, cs, ce, X, S, E, P, out, s)
               : run_mix<__nv_bfloat16, false>(c, cs, ce, X, S, E, P, out, s);
  return vec ? run_mix<__half, true>(c, cs, ce, X, S, E, P, out, s) : run_mix<__half, false>(c, cs, ce, X, S, E, P, out, s);
}

int64_t mix_dcoeff_work_bytes(int S, int E, int64_t P) {
  const int64_t share = dcoeff_share(S, E, P);
  return (P + share - 1) / share * S * E * 4;
}

cudaError_t launch_mix_dcoeff(const void* dW, const void* X, int S, int E, int64_t P, int dtype, float* part,
                              float* out, cudaStream_t s) {
  const bool vec = P % 4 == 0;
  if (dtype == kDtypeF32)
    return vec ? run_dcoeff<float, true>(dW, X, S, E, P, part, out, s)
               : run_dcoeff<float, false>(dW, X, S, E, P, part, out, s);
  if (dtype == kDtypeBf16)
    return vec ? run_dcoeff<__nv_bfloat16, true>(dW, X, S, E, P, part, out, s)
               : run_dcoeff<__nv_bfloat16, false>(dW, X, S, E, P, part, out, s);
  return vec ? run_dcoeff<__half, true>(dW, X, S, E, P, part, out, s)
             : run_dcoeff<__half, false>(dW, X, S, E, P, part, out, s);
}

}  // namespace fuma
