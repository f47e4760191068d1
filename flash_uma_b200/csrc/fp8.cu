// Block-scaled e4m3 operands of the fp8 dense maps (the products are in grouped.cu).
//
// A block of 128 values (activations: along a row; weights: 128 x 128) is stored as e4m3 codes times a
// scale, the smallest power of two 2^k, k >= -126, with max|x| / 2^k <= 448, the largest e4m3 number. A
// power of two makes x / scale exact, so each value is rounded once, to nearest even, and the
// codes do not depend on how a division rounds; it costs at most one bit of the exponent range
// of e4m3 and nothing of its precision. A block that holds a value that is not finite gets the scale
// NaN, which makes every result that depends on it NaN.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "grouped.cuh"
#include "kernels.h"

namespace fuma {

namespace {

// (scale, 1 / scale) from the largest magnitude's bits. amax = (1 + m) 2^e: 448 = 1.75 2^8, so
// k = e - 8, one more if 1 + m > 1.75 (m's 23 bits above 0x600000).
__device__ __forceinline__ float2 block_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return make_float2(__uint_as_float(0x7fc00000u), 0.0f);
  int k = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  if (k < -126) k = -126;
  return make_float2(__uint_as_float((uint32_t)(k + 127) << 23), __uint_as_float((uint32_t)(127 - k) << 23));
}

__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ void load8(const void* x, int64_t i, int dtype, float (&v)[8]) {
  if (dtype == kDtypeF32) {
    const float4 a = ld4_stream(static_cast<const float*>(x) + i), b = ld4_stream(static_cast<const float*>(x) + i + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
  const uint4 u = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + i));
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float2 f;
    if (dtype == kDtypeBf16) {
      __nv_bfloat162 h;
      memcpy(&h, &w[k], 4);
      f = __bfloat1622float2(h);
    } else {
      __half2 h;
      memcpy(&h, &w[k], 4);
      f = __half22float2(h);
    }
    v[2 * k] = f.x;
    v[2 * k + 1] = f.y;
  }
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

}  // namespace

// Rows x [T, K] -> codes [T, ldq] and scales [ceil(K / 128)][T] (block-major: the 128 rows of a GEMM
// tile read theirs as one run). Half a warp takes one block of one row, 8 values a lane; a
// thread block takes 16 rows of one k-block at a time, so scales leave as 64-byte runs. Columns
// [K, ldq) get zero codes. One pass: 2 (4) bytes read, 1 written per value.
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void* __restrict__ x, int64_t ldx, int dtype,
                                                            int64_t T, int K, uint8_t* __restrict__ codes, int64_t ldq,
                                                            float* __restrict__ scales) {
  const int l = threadIdx.x & 15, hrow = threadIdx.x >> 4;
  const int kblocks = (K + 127) / 128;
  const int64_t units = (T + 15) / 16 * kblocks;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t row = u / kblocks * 16 + hrow;
    const int kb = (int)(u % kblocks), k = kb * 128 + l * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row < T && k < K) load8(x, row * ldx + k, dtype, v);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(kFull, m, o));
    const float2 s = block_scale(m);
    if (row < T) {
      if (k < ldq) {
        uint2 q = make_uint2(0u, 0u);
        if (s.y != 0.0f) {
          q.x = e4m3x2(v[0] * s.y, v[1] * s.y) | (e4m3x2(v[2] * s.y, v[3] * s.y) << 16);
          q.y = e4m3x2(v[4] * s.y, v[5] * s.y) | (e4m3x2(v[6] * s.y, v[7] * s.y) << 16);
        }
        *reinterpret_cast<uint2*>(codes + row * ldq + k) = q;
      }
      if (l == 0) scales[(int64_t)kb * T + row] = s.x;
    }
  }
}

// Weights w [G, N, K] fp32 -> codes [G, N, ldq], scales [G][ceil(N/128)][ceil(K/128)], and the same of
// the transposed matrices [G, K, ldt] (the input gradient's operand; blocks of 128 x 128 transpose
// onto themselves, so both hold the same values). One thread block per 128 x 128 block, run once per weight.
__global__ void __launch_bounds__(256) quantize_weight_kernel(const float* __restrict__ w, int N, int K,
                                                              uint8_t* __restrict__ codes, int64_t ldq,
                                                              float* __restrict__ scales, uint8_t* __restrict__ codes_t,
                                                              int64_t ldt, float* __restrict__ scales_t) {
  __shared__ uint32_t wmax[8];
  __shared__ uint8_t tile[128][132];
  const int kb = blockIdx.x, nb = blockIdx.y, g = blockIdx.z;
  const int c = threadIdx.x & 127, r0 = threadIdx.x >> 7;
  const int64_t base = (int64_t)g * N * K;
  uint32_t m = 0;
  for (int r = r0; r < 128; r += 2) {
    const int n = nb * 128 + r, k = kb * 128 + c;
    if (n < N && k < K) m = max(m, abs_bits(w[base + (int64_t)n * K + k]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(kFull, m, o));
  if ((threadIdx.x & 31) == 0) wmax[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, wmax[i]);
  const float2 s = block_scale(m);
  for (int r = r0; r < 128; r += 2) {
    const int n = nb * 128 + r, k = kb * 128 + c;
    const float v = (n < N && k < K && s.y != 0.0f) ? w[base + (int64_t)n * K + k] * s.y : 0.0f;
    const uint8_t q = (uint8_t)(e4m3x2(v, 0.0f) & 0xFFu);
    tile[r][c] = q;
    if (n < N && k < ldq) codes[((int64_t)g * N + n) * ldq + k] = q;
  }
  __syncthreads();
  for (int r = r0; r < 128; r += 2) {
    const int k = kb * 128 + r, n = nb * 128 + c;
    if (k < K && n < ldt) codes_t[((int64_t)g * K + k) * ldt + n] = tile[c][r];
  }
  if (threadIdx.x == 0) {
    scales[((int64_t)g * gridDim.y + nb) * gridDim.x + kb] = s.x;
    scales_t[((int64_t)g * gridDim.x + kb) * gridDim.y + nb] = s.x;
  }
}

void launch_quantize_rows(const void* x, int64_t ldx, int dtype, int64_t T, int K, void* codes, int64_t ldq,
                          float* scales, cudaStream_t s) {
  const int64_t units = (T + 15) / 16 * ((K + 127) / 128);
  quantize_rows_kernel<<<grid_resident(quantize_rows_kernel, 256, units, 1), 256, 0, s>>>(
      x, ldx, dtype, T, K, static_cast<uint8_t*>(codes), ldq, scales);
}

void launch_quantize_weight(const float* w, int G, int N, int K, void* codes, int64_t ldq, float* scales,
                            void* codes_t, int64_t ldt, float* scales_t, cudaStream_t s) {
  quantize_weight_kernel<<<dim3((unsigned)((K + 127) / 128), (unsigned)((N + 127) / 128), (unsigned)G), 256, 0, s>>>(
      w, N, K, static_cast<uint8_t*>(codes), ldq, scales, static_cast<uint8_t*>(codes_t), ldt, scales_t);
}

}  // namespace fuma
