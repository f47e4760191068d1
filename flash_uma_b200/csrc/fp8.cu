// Block-scaled e4m3 operands of the fp8 dense maps (the products are in grouped.cu).
//
// A block of 128 values (activations: along a row; weights: 128 x 128) is stored as e4m3 codes times a
// scale, the smallest power of two 2^k, k >= -126, with max|x| / 2^k <= 448, the largest e4m3 number. A
// power of two makes x / scale exact, so each value is rounded once, to nearest even, and the
// codes do not depend on how a division rounds; it costs at most one bit of the exponent range
// of e4m3 and nothing of its precision. A block that holds a value that is not finite gets the scale
// NaN, which makes every result that depends on it NaN.
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

// two values to e4m3, nearest even, a in the low byte
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  uint16_t q;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(q) : "f"(b), "f"(a));
  return q;
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

}  // namespace

// Rows x [T, K] -> codes [T, ldq] and scales [ceil(K / 128)][T] (block-major: the 128 rows of a GEMM
// tile read theirs as one run). 16 lanes (fp32; 16-bit types: 8) take one block of one row with two 16-byte loads each
// and kQRows such blocks at a time, all loaded before the first reduction; blocks follow one another along the rows, so
// a thread block reads a run of memory. 16-bit types find the largest magnitude on packed pairs. Columns [K, ldq) get
// zero codes. One pass: 2 (4) bytes read, 1 written per value. Bound by HBM: 120,000 x 1024 bf16, 0.37 GB, in
// 62 us (5.9 TB/s), fp32, 0.62 GB, in 99 us (6.2 TB/s).
// kVec: rows 16-byte aligned.
template <int kDtype, int kQRows, bool kVec>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void* __restrict__ x, int64_t ldx, int64_t T, int K,
                                                            uint8_t* __restrict__ codes, int64_t ldq,
                                                            float* __restrict__ scales) {
  constexpr bool kF32 = kDtype == kDtypeF32;
  constexpr int kLanes = kF32 ? 16 : 8, kVals = 128 / kLanes, kUnits = 256 / kLanes;
  const int l = threadIdx.x % kLanes, h = threadIdx.x / kLanes;
  const uint32_t kblocks = (uint32_t)(K + 127) / 128;
  const int64_t units = T * kblocks;
  for (int64_t u0 = (int64_t)blockIdx.x * (kUnits * kQRows); u0 < units; u0 += (int64_t)gridDim.x * (kUnits * kQRows)) {
    const int64_t base = u0 / kblocks;
    const uint32_t rest = (uint32_t)(u0 - base * kblocks) + h;
    uint4 raw[kQRows][2];
    uint32_t drow[kQRows];
    int kb[kQRows];
#pragma unroll
    for (int i = 0; i < kQRows; ++i) {
      const uint32_t v = rest + kUnits * i;
      drow[i] = v / kblocks;
      kb[i] = (int)(v - drow[i] * kblocks);
      const int k = kb[i] * 128 + l * kVals;
      raw[i][0] = raw[i][1] = make_uint4(0u, 0u, 0u, 0u);
      if (!kVec) {
        if (base + drow[i] < T && k < K) {
          constexpr int kSize = kF32 ? 4 : 2;
          uint8_t b[32];
          const uint8_t* src = static_cast<const uint8_t*>(x) + ((base + drow[i]) * ldx + k) * kSize;
#pragma unroll
          for (int j = 0; j < kVals; ++j) {
            if constexpr (kF32) {
              const uint32_t e = k + j < K ? *reinterpret_cast<const uint32_t*>(src + 4 * j) : 0u;
              memcpy(b + 4 * j, &e, 4);
            } else {
              const uint16_t e = k + j < K ? *reinterpret_cast<const uint16_t*>(src + 2 * j) : (uint16_t)0;
              memcpy(b + 2 * j, &e, 2);
            }
          }
          memcpy(raw[i], b, 32);
        }
      } else if (base + drow[i] < T) {   // K is a multiple of 8: a 16-byte load is all inside or all outside
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(x) +
                                                        ((base + drow[i]) * ldx + k) * (kF32 ? 4 : 2));
        if (k < K) raw[i][0] = __ldcs(p);
        if (k + kVals / 2 < K) raw[i][1] = __ldcs(p + 1);
      }
    }
#pragma unroll
    for (int i = 0; i < kQRows; ++i) {
      const uint32_t w[8] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w,
                             raw[i][1].x, raw[i][1].y, raw[i][1].z, raw[i][1].w};
      uint32_t m = 0;
      if constexpr (kF32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, w[j] & 0x7fffffffu);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) asm("max.u16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(w[j] & 0x7fff7fffu));
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) {
        const uint32_t n = __shfl_xor_sync(kFull, m, o);
        if constexpr (kF32) m = max(m, n);
        else asm("max.u16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(n));
      }
      if constexpr (!kF32) {
        m = max(m & 0xffffu, m >> 16);
        if constexpr (kDtype == kDtypeBf16) m <<= 16;
        else m = __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
      }
      const float2 s = block_scale(m);
      const int64_t row = base + drow[i];
      const int k = kb[i] * 128 + l * kVals;
      if (row < T) {
        if (k < ldq) {
          uint32_t q[kVals / 4];
#pragma unroll
          for (int j = 0; j < kVals / 4; ++j) q[j] = 0u;
          if (s.y != 0.0f) {
            float f[kVals];
            if constexpr (kF32) {
#pragma unroll
              for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(w[j]);
            } else if constexpr (kDtype == kDtypeBf16) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                f[2 * j] = __uint_as_float(w[j] << 16);
                f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
              }
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                __half2 v2;
                memcpy(&v2, &w[j], 4);
                const float2 v = __half22float2(v2);
                f[2 * j] = v.x;
                f[2 * j + 1] = v.y;
              }
            }
#pragma unroll
            for (int j = 0; j < kVals / 4; ++j)
              q[j] = e4m3x2(f[4 * j] * s.y, f[4 * j + 1] * s.y) | (e4m3x2(f[4 * j + 2] * s.y, f[4 * j + 3] * s.y) << 16);
          }
          uint8_t* out = codes + row * ldq + k;
          if constexpr (kF32) *reinterpret_cast<uint2*>(out) = make_uint2(q[0], q[1]);
          else *reinterpret_cast<uint4*>(out) = make_uint4(q[0], q[1], q[2], q[3]);
        }
        if (l == 0) scales[(int64_t)kb[i] * T + row] = s.x;
      }
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

template <int kDtype, int kQRows, bool kVec>
static void run_quantize_rows(const void* x, int64_t ldx, int64_t T, int K, void* codes, int64_t ldq, float* scales,
                              cudaStream_t s) {
  const int64_t units = T * ((K + 127) / 128);
  auto kern = quantize_rows_kernel<kDtype, kQRows, kVec>;
  kern<<<grid_resident(kern, 256, units, (kDtype == kDtypeF32 ? 16 : 32) * kQRows), 256, 0, s>>>(
      x, ldx, T, K, static_cast<uint8_t*>(codes), ldq, scales);
}

template <int kDtype>
static void any_quantize_rows(const void* x, int64_t ldx, int64_t T, int K, void* codes, int64_t ldq, float* scales,
                              cudaStream_t s) {
  // few rows: one block per lane group, so that more thread blocks share the work (1,000 x 512 bf16: 2.0 us, with four
  // 3.0; 120,000 x 1024: 64.7, with four 62.6)
  const bool few = T * K < (int64_t)4 << 20, vec = ldx % 8 == 0 && K % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  auto run = vec ? (few ? run_quantize_rows<kDtype, 1, true> : run_quantize_rows<kDtype, 4, true>)
                 : run_quantize_rows<kDtype, 1, false>;
  run(x, ldx, T, K, codes, ldq, scales, s);
}

void launch_quantize_rows(const void* x, int64_t ldx, int dtype, int64_t T, int K, void* codes, int64_t ldq,
                          float* scales, cudaStream_t s) {
  auto run = dtype == kDtypeF32 ? any_quantize_rows<kDtypeF32>
             : dtype == kDtypeBf16 ? any_quantize_rows<kDtypeBf16> : any_quantize_rows<kDtypeF16>;
  run(x, ldx, T, K, codes, ldq, scales, s);
}

void launch_quantize_weight(const float* w, int G, int N, int K, void* codes, int64_t ldq, float* scales,
                            void* codes_t, int64_t ldt, float* scales_t, cudaStream_t s) {
  quantize_weight_kernel<<<dim3((unsigned)((K + 127) / 128), (unsigned)((N + 127) / 128), (unsigned)G), 256, 0, s>>>(
      w, N, K, static_cast<uint8_t*>(codes), ldq, scales, static_cast<uint8_t*>(codes_t), ldt, scales_t);
}

}  // namespace fuma
