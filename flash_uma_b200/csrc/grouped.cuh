// Arguments shared by the grouped dense maps (grouped.cu), the fp8 quantisation (fp8.cu), the
// expert mix (mix.cu) and the C ABI.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

namespace fuma {

constexpr int kMaxGroups = 4096;
constexpr int kDtypeF32 = 0, kDtypeBf16 = 1, kDtypeF16 = 2;
constexpr int kErrOffsets = 64;    // group offsets that decrease or leave [0, T]

// 8 consecutive values of a type, 16-byte aligned, loaded first and converted later: kernels that keep several
// loads in flight take the type as a template argument (a branch on it between the loads makes each wait for the last).
template <int kDtype>
struct Raw8 {
  uint4 w[kDtype == kDtypeF32 ? 2 : 1];
  __device__ __forceinline__ void zero() {
    for (auto& u : w) u = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void load(const void* x, int64_t i) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(x) + i * (kDtype == kDtypeF32 ? 4 : 2));
    w[0] = __ldcs(p);
    if constexpr (kDtype == kDtypeF32) w[1] = __ldcs(p + 1);
  }
  __device__ __forceinline__ void load_some(const void* x, int64_t i, int n) {   // any alignment, n <= 8 values
    constexpr int kSize = kDtype == kDtypeF32 ? 4 : 2;
    uint8_t b[8 * kSize];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (kSize == 4) {
        const uint32_t v = k < n ? static_cast<const uint32_t*>(x)[i + k] : 0u;
        memcpy(b + 4 * k, &v, 4);
      } else {
        const uint16_t v = k < n ? static_cast<const uint16_t*>(x)[i + k] : (uint16_t)0;
        memcpy(b + 2 * k, &v, 2);
      }
    }
    memcpy(w, b, sizeof(b));
  }
  __device__ __forceinline__ void to_f32(float (&v)[8]) const {
    if constexpr (kDtype == kDtypeF32) {
      memcpy(v, w, 32);
    } else {
      const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float2 f;
        if constexpr (kDtype == kDtypeBf16) {
          __nv_bfloat162 h;
          memcpy(&h, &u[k], 4);
          f = __bfloat1622float2(h);
        } else {
          __half2 h;
          memcpy(&h, &u[k], 4);
          f = __half22float2(h);
        }
        v[2 * k] = f.x;
        v[2 * k + 1] = f.y;
      }
    }
  }
};

// kind: 0 bf16 / fp16 (dtype), 1 two fp16 planes of fp32 (split_blocks), 2 e4m3. Leading dimensions in elements.
struct GroupedOperands {
  const void* A;
  const void* B;
  int64_t lda, ldb;
  int kind, dtype;
};

struct GroupedArgs {
  const int64_t* offsets;   // [G + 1], device
  int G;
  int64_t T;                // rows of the ragged operand(s)
  int M, N, K;              // row maps: N output columns, contraction K. Weight gradient: dW is [G, M, N].
  void* C;                  // contiguous
  int out_dtype;
  const void* bias;         // [N] or [G, N] or null
  int bias_rows, bias_dtype;
  // fp8: scale_a [ceil(K / 128)][T], scale_b [G][blocks_n][ceil(K / 128)]. Planes: of the row operands
  // [column blocks][scale_slots], of W [G][ceil(N / 128)][ceil(K / 128)] in the forward's terms.
  const float* scale_a;
  const float* scale_b;
  int blocks_n;             // 128-column blocks of the output
  int64_t scale_slots;
  // Weight gradient: fp32 matrices of the parts of groups longer than cap blocks of 128 rows. Such a group that starts in
  // block A (of absolute rows) and has b > cap blocks takes slots floor(2 A / cap) + part, part < q = ceil(b / cap). The next
  // such group starts in block A + b - 1 or later, so its first slot is at least floor(2 (b - 1) / cap) >= 2 (q - 1) >= q
  // further on. All slots are below 2 (T / 128) / cap + 2.
  void* work;
  int* err;
  // set by the launcher
  int bn, tiles_m, tiles_n, cap, ldw, span, box_b, wide_a, wide_b;
  uint32_t mma_format;
};

int launch_grouped_rows(const GroupedOperands& o, GroupedArgs p, bool transposed, int* err, cudaStream_t s);
int launch_grouped_wgrad(const GroupedOperands& o, GroupedArgs p, int* err, cudaStream_t s);
int64_t grouped_wgrad_work_bytes(int64_t T, int M, int N, int dtype);
int64_t grouped_colsum_work_bytes(int64_t T, int N, int groups);
cudaError_t launch_grouped_colsum(const void* x, int64_t ld, int dtype, const int64_t* off, int G, bool shared,
                                  int64_t T, int N, float* part, void* out, cudaStream_t s);
// Two fp16 planes [2][rows][cols rounded up to 8] and their block scales: of ragged rows (mat_rows 0)
// [ceil(cols / 128)][split_slots],
// of matrices of mat_rows rows [matrices][ceil(mat_rows / 128)][ceil(cols / 128)].
int64_t split_slots(int64_t rows, int G);
void launch_split_blocks(const float* x, int64_t ldx, int64_t rows, int cols, const int64_t* off, int G, int mat_rows,
                         int64_t T, void* out, float* scales, cudaStream_t s);

// 16-bit rows copied to a pitch of ldo (a multiple of 8) elements; see the kernel.
void launch_pad_rows(const void* x, int64_t ldx, int64_t rows, int cols, void* out, int64_t ldo, const int64_t* off,
                     int mat_rows, int64_t T, cudaStream_t s);

void launch_quantize_rows(const void* x, int64_t ldx, int dtype, int64_t T, int K, void* codes, int64_t ldq,
                          float* scales, cudaStream_t s);
void launch_quantize_weight(const float* w, int G, int N, int K, void* codes, int64_t ldq, float* scales,
                            void* codes_t, int64_t ldt, float* scales_t, cudaStream_t s);

// out[s, p] = sum_e c[s * cs + e * ce] X[e, p]
cudaError_t launch_mix(const float* c, int64_t cs, int64_t ce, const void* X, int S, int E, int64_t P, int dtype,
                       void* out, int* err, cudaStream_t s);
int mix_bwd_launches(int S, int E, int dtype, bool dc, bool dX);   // kernels of a launch_mix_bwd
int64_t mix_bwd_work_bytes(int S, int E, int64_t P, int dtype);
// dc and dX (either may be null) from dW; part: mix_bwd_work_bytes when dc is asked for
cudaError_t launch_mix_bwd(const float* c, int64_t cs, int64_t ce, const void* dW, const void* X, int S, int E, int64_t P,
                           int dtype, float* dc, void* dX, double* part, int* err, cudaStream_t s);

}  // namespace fuma
