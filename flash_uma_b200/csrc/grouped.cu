// Dense maps over ragged row groups on the tcgen05 tensor cores: row t of group g goes through
// matrix g. Groups are the row ranges [offsets[g], offsets[g + 1]) of the row-major operands;
// offsets live on the device, so no launch waits for the host to know them.
//
//   forward      Y[t, n]   = sum_k X[t, k] W[g, n, k] (+ b[n] or b[g, n])
//   input grad   dX[t, k]  = sum_n dY[t, n] W[g, n, k]
//   weight grad  dW[g,n,k] = sum_{t in g} dY[t, n] X[t, k]
//
// One persistent kernel covers the three: a work item is a 128 x BN output tile, operand "A"
// supplies its 128 rows (the MMA's M side) and "B" its BN <= 256 columns (the N side). The
// operands are read where they lie: W of the input gradient and both operands of the weight
// gradient are contiguous along the tile and not along the contraction ("MN-major"), which the
// shared-memory descriptors express, so nothing is transposed in memory.
//
// Element types (kKind):
//   kHalf    bf16 or fp16 operands, one kind::f16 product per 16 elements of the contraction.
//   kPlanes  fp32 operands as three bf16 planes x = p0 + p1 + p2 (round to nearest each; 24
//            bits, the whole fp32 exponent range, so no value needs a scale or is refused).
//            Six products: p0 q0 in one accumulator; p0 q1, p1 q0, p1 q1, p0 q2, p2 q0 in a
//            second one, so that the full-size sum takes one truncating addition per 16
//            elements; what is dropped (p1 q2 and below) is 2^-24 of a product.
//   kFp8     e4m3 operands with fp32 scales: sA[kb][row] for each row and block kb of 128 along the
//            contraction, sB[g][n / 128][kb] for each 128 x 128 block of W.
//
// Accumulation: the tensor core truncates each addition to its fp32 accumulator, which drifts over
// long sums, and fp8 products of different blocks carry different scales. So TMEM holds the
// sum of one SEGMENT of the contraction (kHalf: 1024 elements, kPlanes: 128, kFp8: one block of
// 128); eight epilogue warps add each segment to fp32 registers, rounded to nearest and with the
// fp8 scales, while the MMAs of the next segment run in the other TMEM buffer (kPlanes fills
// TMEM with one buffer of 2 x 256 columns, and the drain of 512 columns per 6,144 cycles of MMA
// is exposed).
//
// Structure: 384 threads, one CTA per SM. Warp 0 loads operand tiles by TMA into a ring; warp 1
// allocates TMEM, and its lane 0 issues the MMAs; warps 4-11 are the epilogue. Every wait is bounded.
#include <cstdio>

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "grouped.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace fuma {

namespace {

constexpr int kBM = 128;
constexpr int kMaxBN = 256;
constexpr int kGThreads = 384;      // one control warpgroup (warps 0, 1 work), two epilogue warpgroups
constexpr int kEpiWarps = 8, kEpiWarp0 = 4;
// registers per thread: 384 x 168 at launch, moved to the epilogue (128 x (72 + 216 + 216) in all)
constexpr int kCtrlRegs = 72, kEpiRegs = 216;
constexpr int kHalf = 0, kPlanes = 1, kFp8 = 2;
constexpr int kModeFwd = 0, kModeDx = 1, kModeDw = 2;

template <int kKind>
struct GSmem {
  static constexpr int kP = kKind == kPlanes ? 3 : 1;               // planes per operand
  static constexpr int kElem = kKind == kFp8 ? 1 : 2;               // bytes per element
  static constexpr int kBK = kKind == kFp8 ? 128 : kKind == kPlanes ? 32 : 64;
  static constexpr int kRowBytes = kBK * kElem;                     // K-major tile row: 128 B, kPlanes 64 B
  static constexpr int kA = kBM * kRowBytes;                        // one plane of the A tile
  static constexpr int kB = kMaxBN * kRowBytes;
  static constexpr int kStage = kP * (kA + kB);                     // 48 KB; kPlanes 72 KB
  static constexpr int kStages = kKind == kPlanes ? 2 : 4;
  static constexpr int kStaging = kEpiWarps * 2048;
  static constexpr int kPrefix = (kMaxGroups + 1) * 4 + 60;         // 16-byte multiple
  static constexpr int kBytes = kStages * kStage + kStaging + 512 /*barriers*/ + kPrefix + 1024 /*alignment*/;
  static_assert(kBytes <= 227 * 1024, "shared memory plan exceeds 227 KB");
  static constexpr int kSegBlocks = kKind == kHalf ? 16 : kKind == kPlanes ? 4 : 1;   // k-blocks per segment
  static constexpr int kAccCols = kP == 3 ? 2 * kMaxBN : kMaxBN;    // main (+ cross)
  static constexpr int kBufs = 512 / kAccCols;
};

// MN-major operand, 128-byte swizzle: a tile is chunks of 64 (16-bit) elements along the tile
// dimension, each chunk a run of 128-byte rows along the contraction. Chunks are `chunk` bytes apart
// (leading byte offset), groups of 8 contraction rows 1024 B apart (stride byte offset).
__device__ __forceinline__ uint64_t smem_desc_mn128(uint32_t addr, uint32_t chunk) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)(chunk >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}

// K-major operand, 64-byte swizzle: 8-row groups 512 B apart.
__device__ __forceinline__ uint64_t smem_desc_k64(uint32_t addr) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)1u << 16;
  d |= (uint64_t)(512u >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)4u << 61;
  return d;
}

template <bool kF8>
__device__ __forceinline__ void mma_issue(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (kF8)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

// (x: contiguous, y: rows, z: matrix, w: plane)
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(0), "r"(smem_u32(bar))
      : "memory");
}

// Group g's start, held inside [0, T] whatever the caller's array says; no array: one group of all rows.
__device__ __forceinline__ int64_t group_at(const int64_t* off, int g, int64_t T) {
  if (!off) return g ? T : 0;
  const int64_t o = off[g];
  return o < 0 ? 0 : o > T ? T : o;
}
__device__ __forceinline__ int64_t group_len(const int64_t* off, int g, int64_t T) {
  const int64_t n = group_at(off, g + 1, T) - group_at(off, g, T);
  return n > 0 ? n : 0;
}

// Work units of a group: 128-row tiles (row maps), or chunks of `chunk` contraction rows (weight
// gradient; a group without rows still has one, which writes zeros).
template <int kMode>
__device__ __forceinline__ int group_units(int64_t len, int chunk) {
  if constexpr (kMode == kModeDw) {
    const int64_t n = (len + chunk - 1) / chunk;
    return n > 0 ? (int)n : 1;
  } else {
    return (int)((len + kBM - 1) / kBM);
  }
}

// The group that unit u belongs to: the last g with prefix[g] <= u.
__device__ __forceinline__ int find_group(const int* prefix, int G, int u) {
  int lo = 0, hi = G;   // prefix[lo] <= u < prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= u) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ uint32_t pack_half(float a, float b, int dtype) {
  uint32_t u;
  if (dtype == kDtypeBf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    memcpy(&u, &h, 4);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    memcpy(&u, &h, 4);
  }
  return u;
}

}  // namespace

// One item's place: group, first row and row count on the M side, first contraction row (weight
// gradient), columns, k-blocks.
struct Item {
  int g, n0, kblocks;
  int64_t row0;     // first A row (row maps) or first contraction row (weight gradient)
  int m0, rows;     // weight gradient: first output row; rows of the tile that exist
  int tail;         // weight gradient: contraction rows of the last k-block (0: none)
  int64_t out;      // element offset of (row 0, column 0) of the tile's matrix in the output
  bool partial;     // weight gradient: goes to the fp32 workspace
};

template <int kMode, int kBK>
__device__ __forceinline__ Item item_at(const GroupedArgs& p, const int* prefix, int item) {
  Item t;
  t.partial = false;
  t.tail = 0;
  if constexpr (kMode == kModeDw) {
    const int tiles = p.tiles_m * p.tiles_n;
    const int u = item / tiles, tile = item - u * tiles;
    t.g = find_group(prefix, p.G, u);
    const int c = u - prefix[t.g];
    const int64_t at = group_at(p.offsets, t.g, p.T), len = group_len(p.offsets, t.g, p.T);
    t.row0 = at + (int64_t)c * p.chunk;
    int64_t n = len - (int64_t)c * p.chunk;
    if (n > p.chunk) n = p.chunk;
    t.kblocks = (int)((n + kBK - 1) / kBK);
    t.tail = (int)(n % kBK);
    t.m0 = (tile / p.tiles_n) * kBM;
    t.n0 = (tile % p.tiles_n) * p.bn;
    t.rows = p.M - t.m0 < kBM ? p.M - t.m0 : kBM;
    t.partial = len > p.chunk;
    const int64_t slot = at / p.chunk + c;   // chunk 0 in the first half of the slots, see grouped.cuh
    t.out = (t.partial ? (c == 0 ? slot : p.slots + slot) : (int64_t)t.g) * p.M * p.N + (int64_t)t.m0 * p.N;
  } else {
    const int mt = item / p.tiles_n;
    t.g = find_group(prefix, p.G, mt);
    const int64_t at = group_at(p.offsets, t.g, p.T);
    const int64_t r = (int64_t)(mt - prefix[t.g]) * kBM;
    const int64_t left = group_len(p.offsets, t.g, p.T) - r;
    t.row0 = at + r;
    t.m0 = 0;
    t.rows = left < kBM ? (int)left : kBM;
    t.n0 = (item - mt * p.tiles_n) * p.bn;
    t.kblocks = (p.K + kBK - 1) / kBK;
    t.out = t.row0 * p.ldc;
  }
  return t;
}

template <int kKind, int kMode>
__global__ void __launch_bounds__(kGThreads, 1)
    grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                        const __grid_constant__ GroupedArgs p) {
  using L = GSmem<kKind>;
  constexpr int kP = L::kP, kBK = L::kBK;
  constexpr bool kAmn = kMode == kModeDw;                 // A contiguous along the tile
  constexpr bool kBmn = kMode != kModeFwd;
  constexpr uint32_t kChunkMn = kP * kBK * 128;           // bytes between 64-element chunks (planes inside)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_c = smem + L::kStages * L::kStage;
  uint64_t* bar_full = reinterpret_cast<uint64_t*>(smem_c + L::kStaging);
  uint64_t* bar_empty = bar_full + L::kStages;
  uint64_t* bar_acc_full = bar_empty + L::kStages;   // [2]
  uint64_t* bar_acc_empty = bar_acc_full + 2;        // [2]
  uint64_t* bar_done = bar_acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* scan = reinterpret_cast<int*>(tmem_slot + 2);   // [kGThreads / 32]
  int* prefix = reinterpret_cast<int*>(smem_c + L::kStaging + 512);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bar_acc_full[b], 1);
      mbar_init(&bar_acc_empty[b], kEpiWarps * 32);
    }
    mbar_init(bar_done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // prefix[g] = work units before group g: a contiguous run of groups per thread, then a scan
  // of the threads' sums
  {
    const int per = (p.G + kGThreads - 1) / kGThreads;
    const int g0 = threadIdx.x * per, g1 = min(p.G, g0 + per);
    int sum = 0;
    int bad = 0;
    for (int g = g0; g < g1; ++g) {
      if (p.offsets) {
        const int64_t a = p.offsets[g], b = p.offsets[g + 1];
        bad |= a < 0 || b < a || b > p.T;
      }
      sum += group_units<kMode>(group_len(p.offsets, g, p.T), p.chunk);
    }
    // offsets that decrease or leave [0, T]: recorded, and no item runs (every CTA sees the same array)
    bad = __syncthreads_or(bad);
    if (bad && blockIdx.x == 0 && threadIdx.x == 0 && p.err) atomicCAS(p.err, 0, kErrOffsets);
    if (bad) sum = 0;
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kFull, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    int base = incl - sum;
    for (int w = 0; w < warp; ++w) base += scan[w];
    for (int g = g0; g < g1; ++g) {
      prefix[g] = base;
      if (!bad) base += group_units<kMode>(group_len(p.offsets, g, p.T), p.chunk);
    }
    if (g1 == p.G && g0 < g1) prefix[p.G] = base;
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const int items = prefix[p.G] * (kMode == kModeDw ? p.tiles_m * p.tiles_n : p.tiles_n);

  if (warp < kEpiWarp0) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCtrlRegs));
  if (warp == 0) {
    // ---------------- producer
    if (lane == 0) {
      const int b_chunks = (p.bn + 63) / 64;
      const uint32_t bytes = kP * (L::kA + (kBmn ? b_chunks * kBK * 128 : p.bn * L::kRowBytes));
      int it = 0;
      for (int item = blockIdx.x; item < items && !*abort_flag; item += gridDim.x) {
        const Item t = item_at<kMode, kBK>(p, prefix, item);
        for (int kt = 0; kt < t.kblocks; ++kt, ++it) {
          const int s = it % L::kStages;
          if (it >= L::kStages &&
              !mbar_wait(&bar_empty[s], ((it / L::kStages) - 1) & 1, abort_flag, p.err, kErrWaitEmpty))
            break;
          uint8_t* a = smem + s * L::kStage;
          uint8_t* b = a + kP * L::kA;
          mbar_expect_tx(&bar_full[s], bytes);
          if constexpr (kAmn) {
            for (int c = 0; c < kBM / 64; ++c)
              tma_load_4d(a + c * kChunkMn, &tmA, t.m0 + c * 64, (int)t.row0 + kt * kBK, 0, &bar_full[s]);
          } else {
            tma_load_4d(a, &tmA, kt * kBK, (int)t.row0, 0, &bar_full[s]);
          }
          if constexpr (kBmn) {
            const int y = kMode == kModeDw ? (int)t.row0 + kt * kBK : kt * kBK;
            for (int c = 0; c < b_chunks; ++c)
              tma_load_4d(b + c * kChunkMn, &tmB, t.n0 + c * 64, y, kMode == kModeDw ? 0 : t.g, &bar_full[s]);
          } else {
            tma_load_4d(b, &tmB, kt * kBK, t.n0, t.g, &bar_full[s]);
          }
        }
      }
      if (*abort_flag) {
        for (int j = it - 1; j >= 0 && j >= it - L::kStages; --j) {
          for (uint32_t i = 0; i < kWaitLimit && !mbar_try(&bar_full[j % L::kStages], (j / L::kStages) & 1); ++i) {
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issue
    const uint32_t fmt = p.mma_format;   // operand format bits of the instruction descriptor
    const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (kAmn ? 1u << 15 : 0u) | (kBmn ? 1u << 16 : 0u) |
                           ((uint32_t)(p.bn >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
    int it = 0, seg = 0;
    bool ok = true;
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const Item t = item_at<kMode, kBK>(p, prefix, item);
      for (int kt = 0; kt < t.kblocks && ok; ++kt, ++it) {
        const int s = it % L::kStages, buf = seg % L::kBufs;
        const bool first = kt % L::kSegBlocks == 0;
        if (first && seg >= L::kBufs)
          ok = mbar_wait(&bar_acc_empty[buf], ((seg / L::kBufs) - 1) & 1, abort_flag, p.err, kErrWaitAccEmpty);
        ok = ok && mbar_wait(&bar_full[s], (it / L::kStages) & 1, abort_flag, p.err, kErrWaitFull);
        ok = __all_sync(kFull, ok);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint8_t* sa = smem + s * L::kStage;
        uint8_t* sb = sa + kP * L::kA;
        int steps = kBK * L::kElem / 32;
        if constexpr (kMode == kModeDw) {
          // the last k-block of a group ends inside the tile: the rows behind it belong to the next
          // group (whatever they hold must not count). Only whole steps of 16 rows run, and
          // the rest of the last one is cleared in both operands (0 x inf would be NaN).
          if (kt == t.kblocks - 1 && t.tail) {
            steps = (t.tail + 15) / 16;
            const int dead = steps * 16 - t.tail;
            const int chunks = kBM / 64 * kP, chunks_b = (p.bn + 63) / 64 * kP;
            for (int i = lane; i < (chunks + chunks_b) * dead * 8; i += 32) {
              const int c = i / (dead * 8), r = (i / 8) % dead, j = i % 8;
              uint8_t* base = c < chunks ? sa + c * (kBK * 128) : sb + (c - chunks) * (kBK * 128);
              *reinterpret_cast<uint4*>(base + (t.tail + r) * 128 + j * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
        }
        if (lane == 0) {
          const uint32_t a0 = smem_u32(sa), b0 = smem_u32(sb);
          const uint32_t acc_main = tmem + (uint32_t)(buf * L::kAccCols), acc_cross = acc_main + kMaxBN;
          auto desc_a = [&](int plane, int kk) {
            if constexpr (kAmn) return smem_desc_mn128(a0 + plane * (kBK * 128) + kk * 2048, kChunkMn);
            else if constexpr (L::kRowBytes == 64) return smem_desc_k64(a0 + plane * L::kA + kk * 32);
            else return smem_desc_sw128(a0 + kk * 32);
          };
          auto desc_b = [&](int plane, int kk) {
            if constexpr (kBmn) return smem_desc_mn128(b0 + plane * (kBK * 128) + kk * 2048, kChunkMn);
            else if constexpr (L::kRowBytes == 64) return smem_desc_k64(b0 + plane * (p.bn * L::kRowBytes) + kk * 32);
            else return smem_desc_sw128(b0 + kk * 32);
          };
          for (int kk = 0; kk < steps; ++kk) {
            const uint32_t acc = (first && kk == 0) ? 0u : 1u;
            mma_issue<kKind == kFp8>(acc_main, desc_a(0, kk), desc_b(0, kk), idesc, acc);
            if constexpr (kKind == kPlanes) {
              mma_issue<false>(acc_cross, desc_a(0, kk), desc_b(1, kk), idesc, acc);
              mma_issue<false>(acc_cross, desc_a(1, kk), desc_b(0, kk), idesc, 1u);
              mma_issue<false>(acc_cross, desc_a(1, kk), desc_b(1, kk), idesc, 1u);
              mma_issue<false>(acc_cross, desc_a(0, kk), desc_b(2, kk), idesc, 1u);
              mma_issue<false>(acc_cross, desc_a(2, kk), desc_b(0, kk), idesc, 1u);
            }
          }
          mma_commit(&bar_empty[s]);
          if (kt % L::kSegBlocks == L::kSegBlocks - 1 || kt == t.kblocks - 1) mma_commit(&bar_acc_full[buf]);
        }
        __syncwarp();
        if (kt % L::kSegBlocks == L::kSegBlocks - 1 || kt == t.kblocks - 1) ++seg;
      }
    }
    if (lane == 0) {
      mma_commit(bar_done);
      for (uint32_t i = 0; i < kWaitLimit && !mbar_try(bar_done, 0); ++i) {
      }
    }
    __syncwarp();
  }
  } else {
    // ---------------- epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
    const int q = warp & 3, half = (warp - kEpiWarp0) >> 2;
    uint8_t* stage = smem_c + (warp - kEpiWarp0) * 2048;
    if constexpr (kMode != kModeDw) {
      // rows before the first and behind the last group: zeros
      const int64_t head = group_at(p.offsets, 0, p.T), tail = group_at(p.offsets, p.G, p.T);
      const int vec = p.N * (p.out_dtype == kDtypeF32 ? 4 : 2) / 16;
      const int64_t dead = prefix[p.G] || head == tail ? head + (p.T - tail) : 0, n = dead * vec;
      for (int64_t i = (int64_t)blockIdx.x * (kEpiWarps * 32) + threadIdx.x - kEpiWarp0 * 32; i < n;
           i += (int64_t)gridDim.x * (kEpiWarps * 32)) {
        const int64_t r = i / vec, row = r < head ? r : tail + (r - head);
        uint8_t* c = static_cast<uint8_t*>(p.C) + row * p.ldc * (p.out_dtype == kDtypeF32 ? 4 : 2);
        reinterpret_cast<uint4*>(c)[i - r * vec] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    const int hw = p.bn > 128 ? 128 : (p.bn + 63) / 64 * 32;   // columns of this warp: [half * hw, + hw)
    const int col0 = half * hw;
    int seg = 0;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
      const Item t = item_at<kMode, kBK>(p, prefix, item);
      const int segs = (t.kblocks + L::kSegBlocks - 1) / L::kSegBlocks;
      const int n0 = t.n0 + col0;
      const int ncols = min(min(hw, p.bn - col0), p.N - n0);   // this warp's columns that exist (may be <= 0)
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
      const float* sa = nullptr;
      const float* sb = nullptr;
      float a_next = 1.0f, b_next = 1.0f;
      if constexpr (kKind == kFp8) {
        // the scales of one segment ahead, so their latency hides behind the wait for its MMAs
        const int64_t r = min(t.row0 + q * 32 + lane, p.T - 1);
        sa = p.scale_a + r;
        sb = p.scale_b + ((int64_t)t.g * p.blocks_n + min(n0 / 128, p.blocks_n - 1)) * t.kblocks;
        a_next = sa[0];
        b_next = sb[0];
      }
      bool ok = true;
      for (int sg = 0; sg < segs; ++sg, ++seg) {
        const int buf = seg % L::kBufs;
        const float s_a = a_next, s_b = b_next;   // multiplied after the wait: the loads stay in flight
        if constexpr (kKind == kFp8) {
          const int kb = sg + 1 < segs ? sg + 1 : sg;
          a_next = sa[(int64_t)kb * p.T];
          b_next = sb[kb];
        }
        ok = mbar_wait(&bar_acc_full[buf], (seg / L::kBufs) & 1, abort_flag, p.err, kErrWaitAcc);
        ok = __all_sync(kFull, ok && !*abort_flag);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const float s = s_a * s_b;
        const uint32_t taddr = tmem + (uint32_t)(buf * L::kAccCols + col0) + ((uint32_t)(q * 32) << 16);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c * 32 < ncols) {
            uint32_t r[32];
            tmem_ld32(taddr + c * 32, r);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int u = 0; u < 32; ++u) {
              if constexpr (kKind == kFp8) acc[c * 32 + u] = fmaf(__uint_as_float(r[u]), s, acc[c * 32 + u]);
              else acc[c * 32 + u] += __uint_as_float(r[u]);
            }
            if constexpr (kKind == kPlanes) {
              tmem_ld32(taddr + kMaxBN + c * 32, r);
              asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
              for (int u = 0; u < 32; ++u) acc[c * 32 + u] += __uint_as_float(r[u]);
            }
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive(&bar_acc_empty[buf]);
      }
      if (!ok) break;
      if (ncols <= 0) continue;

      // bias of this warp's columns through the staging area (fp32), added before the one rounding
      if constexpr (kMode == kModeFwd) {
        if (p.bias) {
          const int64_t b0 = (p.bias_rows > 1 ? (int64_t)t.g * p.N : 0) + n0;
          float v[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int c = lane * 4 + u;
            v[u] = 0.0f;
            if (c < ncols) {
              if (p.bias_dtype == kDtypeF32) v[u] = static_cast<const float*>(p.bias)[b0 + c];
              else if (p.bias_dtype == kDtypeBf16) v[u] = __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[b0 + c]);
              else v[u] = __half2float(static_cast<const __half*>(p.bias)[b0 + c]);
            }
          }
          __syncwarp();
          reinterpret_cast<float4*>(stage)[lane] = make_float4(v[0], v[1], v[2], v[3]);
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const float4 b = reinterpret_cast<const float4*>(stage)[c];
            acc[4 * c] += b.x; acc[4 * c + 1] += b.y; acc[4 * c + 2] += b.z; acc[4 * c + 3] += b.w;
          }
        }
      }
      // rows out: 64 bytes of each of the warp's 32 rows at a time through the staging area (16-byte
      // chunk j of row r at j ^ ((r >> 1) & 3)), so a store instruction writes 8 rows x 64 bytes
      const int out_dtype = (kMode == kModeDw && t.partial) ? kDtypeF32 : p.out_dtype;
      uint8_t* out = static_cast<uint8_t*>((kMode == kModeDw && t.partial) ? p.work : p.C);
      const int64_t ld = kMode == kModeDw ? p.N : p.ldc;
      const int rows = t.rows - q * 32;   // of this warp
      const int rr = lane >> 2, jj = lane & 3;
      if (out_dtype == kDtypeF32) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          if (c * 16 < ncols) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<float4*>(stage + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
                  make_float4(acc[c * 16 + 4 * j], acc[c * 16 + 4 * j + 1], acc[c * 16 + 4 * j + 2], acc[c * 16 + 4 * j + 3]);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = i * 8 + rr;
              const float4 v = *reinterpret_cast<const float4*>(stage + r * 64 + ((jj ^ ((r >> 1) & 3)) << 4));
              if (r < rows && c * 16 + jj * 4 < ncols)
                *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + t.out + (q * 32 + r) * ld + n0 + c * 16 + jj * 4) = v;
            }
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c * 32 < ncols) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float* a = acc + c * 32 + 8 * j;
              *reinterpret_cast<uint4*>(stage + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
                  make_uint4(pack_half(a[0], a[1], out_dtype), pack_half(a[2], a[3], out_dtype),
                             pack_half(a[4], a[5], out_dtype), pack_half(a[6], a[7], out_dtype));
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = i * 8 + rr;
              const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 64 + ((jj ^ ((r >> 1) & 3)) << 4));
              if (r < rows && c * 32 + jj * 8 < ncols)
                *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + t.out + (q * 32 + r) * ld + n0 + c * 32 + jj * 8) = v;
            }
          }
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ---- joining the chunks of the weight gradient --------------------------------------------------
// dW[g] = sum over the group's chunks, in order, for groups of more than one chunk. Block row y takes the y-th such
// group (there are at most T / chunk of them), found by a count over all groups: 256 threads with a run each.
__global__ void __launch_bounds__(256) grouped_join_kernel(const __grid_constant__ GroupedArgs p) {
  __shared__ int count[8], found;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int per = (p.G + 255) / 256, g0 = threadIdx.x * per, g1 = min(p.G, g0 + per);
  int n = 0;
  for (int g = g0; g < g1; ++g) n += group_len(p.offsets, g, p.T) > p.chunk;
  int incl = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(kFull, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) count[w] = incl;
  if (threadIdx.x == 0) found = -1;
  __syncthreads();
  int before = incl - n;
  for (int i = 0; i < w; ++i) before += count[i];
  const int y = blockIdx.y;
  if (before <= y && y < before + n) {
    for (int g = g0; g < g1; ++g)
      if (group_len(p.offsets, g, p.T) > p.chunk && before++ == y) found = g;
  }
  __syncthreads();
  const int g = found;
  if (g < 0) return;
  const int64_t at = group_at(p.offsets, g, p.T), len = group_len(p.offsets, g, p.T);
  const int chunks = (int)((len + p.chunk - 1) / p.chunk);
  const int64_t n4 = (int64_t)p.M * p.N / 4, slot = at / p.chunk;
  const float* first = static_cast<const float*>(p.work) + slot * n4 * 4;
  const float* rest = static_cast<const float*>(p.work) + (p.slots + slot) * n4 * 4;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n4; i += (int64_t)gridDim.x * blockDim.x) {
    float4 s = ld4_stream(first + i * 4);
#pragma unroll 4
    for (int c = 1; c < chunks; ++c) s += ld4_stream(rest + (c * n4 + i) * 4);
    const int64_t o = ((int64_t)g * n4 + i) * 4;
    if (p.out_dtype == kDtypeF32)
      st4(static_cast<float*>(p.C) + o, s);
    else
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.C) + o) =
          make_uint2(pack_half(s.x, s.y, p.out_dtype), pack_half(s.z, s.w, p.out_dtype));
  }
}

// ---- bias gradient ------------------------------------------------------------------------------
// db[g, n] = sum of dY[t, n] over the rows of group g, in two steps without atomics. The rows are cut at
// multiples of kSumRows and at the group bounds; the piece of row block b and group g writes its fp32
// sums to slot b + g. Walking the pieces in row order moves on b or g each time, so the slots are
// distinct, and there are at most T / kSumRows + G of them. The second step adds a group's
// pieces in fp64 and rounds once. `shared`: all rows between the first and the last offset count as one group.
constexpr int kSumRows = 128;

__device__ __forceinline__ int64_t sum_bound(const int64_t* off, int g, int G, int64_t T, int shared) {
  return group_at(off, shared ? (g ? G : 0) : g, T);
}

// A block takes the pieces of one row block in 256 columns (8 per lane). Long pieces: the 8 warps share a piece's rows,
// 8 rows in flight each, and join in shared memory. Row blocks cut into many short pieces (many small groups):
// a warp per piece, no joining.
template <int kDtype>
__global__ void __launch_bounds__(256) grouped_colsum_kernel(const void* __restrict__ x, int64_t ld,
                                                             const int64_t* __restrict__ off, int G, int shared,
                                                             int64_t T, int N, float* __restrict__ part) {
  __shared__ float sm[8][256 + 8];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int n = blockIdx.y * 256 + lane * 8;
  const int groups = shared ? 1 : G;
  const int64_t b0 = (int64_t)blockIdx.x * kSumRows, b1 = min(T, b0 + kSumRows);
  auto first_behind = [&](int64_t row) {   // first group that ends behind `row`
    int lo = 0, hi = groups;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (sum_bound(off, mid + 1, G, T, shared) > row) hi = mid; else lo = mid + 1;
    }
    return lo;
  };
  const int g0 = first_behind(b0), g1 = min(groups, first_behind(b1 - 1) + 1);
  const bool short_pieces = g1 - g0 > 4;
  const int step = short_pieces ? 1 : 8, w0 = short_pieces ? 0 : w;
  for (int g = g0 + (short_pieces ? w : 0); g < g1; g += short_pieces ? 8 : 1) {
    const int64_t r0 = max(sum_bound(off, g, G, T, shared), b0), r1 = min(sum_bound(off, g + 1, G, T, shared), b1);
    if (r0 >= r1) continue;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (n < N) {
      for (int64_t r = r0 + w0; r < r1; r += 8 * step) {
        Raw8<kDtype> raw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          raw[i].zero();
          if (r + i * step < r1) raw[i].load(x, (r + i * step) * ld + n);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float v[8];
          raw[i].to_f32(v);
#pragma unroll
          for (int k = 0; k < 8; ++k) s[k] += v[k];
        }
      }
    }
    float* out = part + ((int64_t)blockIdx.x + g) * N;
    if (short_pieces) {
      if (n < N) {
        st4(out + n, make_float4(s[0], s[1], s[2], s[3]));
        st4(out + n + 4, make_float4(s[4], s[5], s[6], s[7]));
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) sm[w][lane * 8 + k] = s[k];
      __syncthreads();
      const int c = blockIdx.y * 256 + threadIdx.x;
      if (c < N) {
        float t = sm[0][threadIdx.x];
#pragma unroll
        for (int k = 1; k < 8; ++k) t += sm[k][threadIdx.x];
        out[c] = t;
      }
      __syncthreads();
    }
  }
}

// Second step. Groups of many pieces (or few groups): a block of 32 warps per group and 32 columns, the warps sharing
// the pieces. Many groups of few pieces: a warp per group.
constexpr int kJoinWarps = 32;
__global__ void __launch_bounds__(32 * kJoinWarps) grouped_colsum_join_kernel(const float* __restrict__ part,
                                                                              const int64_t* __restrict__ off, int G,
                                                                              int shared, int64_t T, int N,
                                                                              void* __restrict__ out, int dtype, bool by_warp) {
  __shared__ double sm[kJoinWarps][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int n = blockIdx.x * 32 + lane, groups = shared ? 1 : G;
  auto store = [&](int g, double t) {
    const int64_t o = (int64_t)g * N + n;
    if (dtype == kDtypeF32) static_cast<float*>(out)[o] = (float)t;
    else if (dtype == kDtypeBf16) static_cast<__nv_bfloat16*>(out)[o] = __double2bfloat16(t);
    else static_cast<__half*>(out)[o] = __double2half(t);
  };
  if (by_warp) {
    for (int g = blockIdx.y * kJoinWarps + w; g < groups; g += gridDim.y * kJoinWarps) {
      const int64_t ga = sum_bound(off, g, G, T, shared), gb = sum_bound(off, g + 1, G, T, shared);
      double s = 0.0;
      if (n < N) {
        if (gb > ga)
#pragma unroll 4
          for (int64_t b = ga / kSumRows; b <= (gb - 1) / kSumRows; ++b) s += (double)part[(b + g) * N + n];
        store(g, s);
      }
    }
    return;
  }
  for (int g = blockIdx.y; g < groups; g += gridDim.y) {
    const int64_t ga = sum_bound(off, g, G, T, shared), gb = sum_bound(off, g + 1, G, T, shared);
    double s = 0.0;
    if (n < N && gb > ga) {
      const int64_t last = (gb - 1) / kSumRows;
#pragma unroll 4
      for (int64_t b = ga / kSumRows + w; b <= last; b += kJoinWarps) s += (double)part[(b + g) * N + n];
    }
    sm[w][lane] = s;
    __syncthreads();
    if (w == 0 && n < N) {
      double t = sm[0][lane];
#pragma unroll
      for (int k = 1; k < kJoinWarps; ++k) t += sm[k][lane];
      store(g, t);
    }
    __syncthreads();
  }
}

// ---- fp32 -> three bf16 planes --------------------------------------------------------------------
// x = p0 + p1 + p2 with p0 = bf16(x), p1 = bf16(x - p0), p2 = bf16(x - p0 - p1); the differences are
// exact in fp32. A value that is not finite keeps p0 and zero residuals. 4 values per thread.
__global__ void __launch_bounds__(256) split_bf16x3_kernel(const float* __restrict__ x, int64_t ldx, int64_t rows,
                                                           int cols, __nv_bfloat16* __restrict__ out) {
  const int c4 = cols / 4;
  const int64_t total = rows * c4, plane = rows * cols;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / c4;
    const int c = (int)(i - r * c4) * 4;
    const float4 v = ld4_stream(x + r * ldx + c);
    const float in[4] = {v.x, v.y, v.z, v.w};
    __nv_bfloat16 p[3][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      // beyond the largest bf16 the rounding would give infinity: keep the value below it in p0
      __nv_bfloat16 h = __float2bfloat16_rn(in[u]);
      if (__hisinf(h) && fabsf(in[u]) <= 3.402823466e38f) h = __float2bfloat16_rz(in[u]);
      const float f0 = __bfloat162float(h);
      const float r1 = fabsf(in[u]) <= 3.402823466e38f ? in[u] - f0 : 0.0f;
      const __nv_bfloat16 m = __float2bfloat16_rn(r1);
      p[0][u] = h;
      p[1][u] = m;
      p[2][u] = __float2bfloat16_rn(r1 - __bfloat162float(m));
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      uint2 u;
      memcpy(&u, p[k], 8);
      *reinterpret_cast<uint2*>(out + k * plane + r * cols + c) = u;
    }
  }
}

// ---- host side --------------------------------------------------------------------------------------

namespace {

template <int kKind, int kMode>
cudaError_t launch_grouped(const CUtensorMap& a, const CUtensorMap& b, const GroupedArgs& p, int64_t max_items,
                           cudaStream_t s) {
  using L = GSmem<kKind>;
  auto kern = grouped_gemm_kernel<kKind, kMode>;
  static thread_local uint64_t configured = 0;  // one bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(configured >> (dev & 63) & 1)) {
    cudaError_t st = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
    if (st != cudaSuccess) return st;
    configured |= uint64_t(1) << (dev & 63);
  }
  const int64_t sms = sm_count();
  const int grid = (int)(max_items < 1 ? 1 : max_items < sms ? max_items : sms);
  kern<<<grid, kGThreads, L::kBytes, s>>>(a, b, p);
  return cudaGetLastError();
}

// Columns per tile: the whole width in even parts of at most 256 (a multiple of 16, so that
// N = 640 runs as 3 x 224 and not as 2 x 256 + 128), and narrower tiles, down to 32, while there
// would be fewer tiles than SMs: a call of a few rows is bound by how many SMs pull its matrices in.
// Measured: see the table in the kernel's comment on small calls.
int pick_bn(int N, int64_t tiles_rows, bool fp8) {
  int bn;
  if (fp8) {
    bn = N > 128 ? 256 : 128;   // whole 128-blocks of the scales
  } else {
    const int parts = (N + kMaxBN - 1) / kMaxBN;
    bn = ((N + parts - 1) / parts + 15) / 16 * 16;
  }
  while (bn > 32 && tiles_rows * ((N + bn - 1) / bn) < sm_count()) {
    const int half = fp8 ? bn / 2 : (bn / 2 + 15) / 16 * 16;
    if (half < 32) break;
    bn = half;
  }
  return bn;
}

}  // namespace

int launch_grouped_rows(const GroupedOperands& o, GroupedArgs p, bool transposed, int* err, cudaStream_t s) {
  const bool fp8 = o.kind == kFp8, planes = o.kind == kPlanes;
  const int esize = fp8 ? 1 : 2, P = planes ? 3 : 1;
  const int bk = fp8 ? 128 : planes ? 32 : 64;
  const int64_t groups = p.G < p.T ? p.G : p.T;
  const int64_t tiles_rows = p.T / kBM + groups;   // upper bound: a partial tile per group
  p.bn = pick_bn(p.N, tiles_rows, fp8);
  p.tiles_n = (p.N + p.bn - 1) / p.bn;
  p.tiles_m = 1;
  p.err = err;
  p.chunk = 0;
  p.mma_format = fp8 ? 0u : (planes || o.dtype == kDtypeBf16) ? 1u : 0u;
  const CUtensorMapDataType dt = fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                 : (planes || o.dtype == kDtypeBf16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                     : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUtensorMapSwizzle ksw = planes ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  CUtensorMap ma, mb;
  // A: [T rows, K], planes T * lda apart
  if (!make_map_4d(&ma, dt, o.A, p.K, p.T, 1, P, o.lda * esize, p.T * o.lda * esize, p.T * o.lda * esize, bk, kBM, P,
                   ksw))
    return -1;
  // W: forward [G, N, K] with K contiguous along the contraction; input gradient [G, K, N] with the
  // output columns contiguous
  const int64_t brows = transposed ? p.K : p.N, bcols = transposed ? p.N : p.K;
  if (!make_map_4d(&mb, dt, o.B, bcols, brows, p.G, P, o.ldb * esize, brows * o.ldb * esize,
                   p.G * brows * o.ldb * esize, transposed ? 64 : bk, transposed ? bk : p.bn, P,
                   transposed ? CU_TENSOR_MAP_SWIZZLE_128B : ksw))
    return -1;
  const int64_t items = tiles_rows * p.tiles_n;
  cudaError_t st;
  if (fp8) st = launch_grouped<kFp8, kModeFwd>(ma, mb, p, items, s);
  else if (planes)
    st = transposed ? launch_grouped<kPlanes, kModeDx>(ma, mb, p, items, s)
                    : launch_grouped<kPlanes, kModeFwd>(ma, mb, p, items, s);
  else
    st = transposed ? launch_grouped<kHalf, kModeDx>(ma, mb, p, items, s)
                    : launch_grouped<kHalf, kModeFwd>(ma, mb, p, items, s);
  return (int)st;
}

// Rows of the contraction per work item of the weight gradient: long groups are cut so that about
// three rounds of tiles fill the SMs, but not below 2048 rows, where writing and joining the fp32
// partial matrices costs as much as the products.
static int wgrad_chunk(int64_t T, int tiles) {
  int64_t c = T * tiles / ((int64_t)148 * 3);
  if (c < 2048) c = 2048;
  if (c > (1 << 20)) c = 1 << 20;
  return (int)((c + 63) / 64 * 64);
}

static int wgrad_bn(int N) {
  const int parts = (N + kMaxBN - 1) / kMaxBN;
  return ((N + parts - 1) / parts + 15) / 16 * 16;
}

static int wgrad_tiles(int M, int N) {
  const int bn = wgrad_bn(N);
  return (M + kBM - 1) / kBM * ((N + bn - 1) / bn);
}

int64_t grouped_wgrad_work_bytes(int64_t T, int M, int N) {
  const int chunk = wgrad_chunk(T, wgrad_tiles(M, N));
  if (T <= chunk) return 0;
  return 2 * (T / chunk + 1) * (int64_t)M * N * 4;
}

int launch_grouped_wgrad(const GroupedOperands& o, GroupedArgs p, int* err, cudaStream_t s) {
  const bool planes = o.kind == kPlanes;
  const int P = planes ? 3 : 1, bk = planes ? 32 : 64;
  p.err = err;
  p.bn = wgrad_bn(p.N);
  p.tiles_n = (p.N + p.bn - 1) / p.bn;
  p.tiles_m = (p.M + kBM - 1) / kBM;
  p.chunk = wgrad_chunk(p.T, p.tiles_m * p.tiles_n);
  p.slots = p.T / p.chunk + 1;
  p.mma_format = (planes || o.dtype == kDtypeBf16) ? 1u : 0u;
  p.ldc = p.N;
  const CUtensorMapDataType dt = (planes || o.dtype == kDtypeBf16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                   : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap ma, mb;
  if (!make_map_4d(&ma, dt, o.A, p.M, p.T, 1, P, o.lda * 2, p.T * o.lda * 2, p.T * o.lda * 2, 64, bk, P,
                   CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_map_4d(&mb, dt, o.B, p.N, p.T, 1, P, o.ldb * 2, p.T * o.ldb * 2, p.T * o.ldb * 2, 64, bk, P,
                   CU_TENSOR_MAP_SWIZZLE_128B))
    return -1;
  const int64_t items = (p.T / p.chunk + p.G) * (int64_t)p.tiles_m * p.tiles_n;
  cudaError_t st = planes ? launch_grouped<kPlanes, kModeDw>(ma, mb, p, items, s)
                          : launch_grouped<kHalf, kModeDw>(ma, mb, p, items, s);
  if (st == cudaSuccess && p.T > p.chunk) {
    const int64_t n4 = (int64_t)p.M * p.N / 4;
    int64_t bx = (n4 + 255) / 256;
    if (bx > 512) bx = 512;
    const int64_t by = p.T / p.chunk < p.G ? p.T / p.chunk : p.G;
    grouped_join_kernel<<<dim3((unsigned)bx, (unsigned)by), 256, 0, s>>>(p);
    st = cudaGetLastError();
  }
  return (int)st;
}

int64_t grouped_colsum_work_bytes(int64_t T, int N, int groups) {
  return ((T + kSumRows - 1) / kSumRows + groups) * N * 4;
}

cudaError_t launch_grouped_colsum(const void* x, int64_t ld, int dtype, const int64_t* off, int G, bool shared,
                                  int64_t T, int N, float* part, void* out, cudaStream_t s) {
  const int groups = shared ? 1 : G;
  if (T > 0) {
    auto kern = dtype == kDtypeF32 ? grouped_colsum_kernel<kDtypeF32>
                : dtype == kDtypeBf16 ? grouped_colsum_kernel<kDtypeBf16> : grouped_colsum_kernel<kDtypeF16>;
    kern<<<dim3((unsigned)((T + kSumRows - 1) / kSumRows), (unsigned)((N + 255) / 256)), 256, 0, s>>>(
        x, ld, off, G, shared, T, N, part);
    const cudaError_t st = cudaGetLastError();
    if (st != cudaSuccess) return st;
  }
  const bool by_warp = groups >= 8 && T / groups < 8 * kSumRows;
  const int gy = by_warp ? (groups + kJoinWarps - 1) / kJoinWarps : groups;
  grouped_colsum_join_kernel<<<dim3((unsigned)((N + 31) / 32), (unsigned)gy), 32 * kJoinWarps, 0, s>>>(
      part, off, G, shared, T, N, out, dtype, by_warp);
  return cudaGetLastError();
}

void launch_split_bf16x3(const float* x, int64_t ldx, int64_t rows, int cols, void* out, cudaStream_t s) {
  split_bf16x3_kernel<<<grid_resident(split_bf16x3_kernel, 256, rows * (cols / 4), 256), 256, 0, s>>>(
      x, ldx, rows, cols, static_cast<__nv_bfloat16*>(out));
}

}  // namespace fuma
