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
//   kSplit   fp32 operands as two fp16 planes of each 128 x 128 block under the block's own power-of-two
//            scale 2^k (largest magnitude to [2^14, 2^15)): x = 2^k (hi + lo), hi = fp16(x / 2^k), lo = fp16(x / 2^k
//            - hi). 22 bits for values down to 2^-18 of the block's largest and 2^-40 of that below, over the
//            whole fp32 range. Three products, hi hi, hi lo, lo hi, in one accumulator. (Three bf16 planes need no scale,
//            but six products and half as much again in operand bytes: 260 us where this takes 162, at 30,000 rows
//            in 32 groups, 1024 -> 512.)
//   kFp8     e4m3 operands with fp32 scales: sA[kb][row] for each row and block kb of 128 along the
//            contraction, sB[g][n / 128][kb] for each 128 x 128 block of W.
//
// Accumulation: the tensor core truncates each addition to its fp32 accumulator, which drifts over
// long sums, and the products of different blocks carry different scales. So TMEM holds the
// sum of one SEGMENT of the contraction (kHalf: 1024 elements, kSplit and kFp8: one block of
// 128); eight epilogue warps add each segment to fp32 registers, rounded to nearest and with the
// block scales, while the MMAs of the next segment run in the other of two TMEM buffers.
//
// CTA pairs (kPair, row maps): two CTAs share a 256 x BN tile; each loads its own 128 rows and half of B's columns, and
// the first issues cta_group::2 MMAs for both. Shared-memory traffic is what bounds the single-CTA tile: per
// 64 elements of the contraction 48 KB go in by TMA and 48 KB out to the MMAs, 768 cycles at 128 B/cycle against 512 of
// MMA; a pair moves 32 KB each way.
//
// Structure: 384 threads, one CTA per SM. Warp 0 loads operand tiles by TMA into a ring; warp 1
// allocates TMEM and issues the MMAs from one elected lane; warp 2 (weight gradient) clears the rows behind a group's end; warp 3
// works out the items ahead of time and hands them to the others through a ring (with every warp doing it, 64-bit
// divisions and dependent loads took 1,000 cycles of each tile's epilogue); warps 4-11 are the epilogue. The MMA
// thread's own instructions count: 512 cycles of MMA per stage leave no room for descriptors built from scratch
// (960 cycles per stage measured), so it adds constants to descriptors made once. Every wait is bounded.
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
constexpr int kCoarse = 256;         // entries of the work prefix in shared memory
constexpr int kGThreads = 384;      // one control warpgroup (warps 0, 1 work), two epilogue warpgroups
constexpr int kEpiWarps = 8, kEpiWarp0 = 4;
// registers per thread: 384 x 168 at launch, moved to the epilogue (128 x (72 + 216 + 216) in all)
constexpr int kCtrlRegs = 72, kEpiRegs = 216;
constexpr int kHalf = 0, kSplit = 1, kFp8 = 2;
constexpr int kModeFwd = 0, kModeDx = 1, kModeDw = 2;

template <int kKind, bool kPair>
struct GSmem {
  static constexpr int kP = kKind == kSplit ? 2 : 1;                // planes per operand
  static constexpr int kElem = kKind == kFp8 ? 1 : 2;               // bytes per element
  static constexpr int kBK = kKind == kFp8 ? 128 : kKind == kSplit ? 32 : 64;
  static constexpr int kRowBytes = kBK * kElem;                     // K-major tile row: 128 B, kSplit 64 B
  static constexpr int kA = kBM * kRowBytes;                        // one plane of the A tile
  static constexpr int kB = (kPair ? kMaxBN / 2 : kMaxBN) * kRowBytes;
  static constexpr int kStage = kP * (kA + kB);                     // 48 KB; a pair 32 KB in each CTA
  static constexpr int kStages = kPair ? 6 : 4;
  static constexpr int kStaging = kEpiWarps * 4096;
  static constexpr int kPrefix = (kCoarse + 1) * 4 + 12;            // a multiple of 16
  static constexpr int kBytes = kStages * kStage + kStaging + 640 /*barriers, items*/ + kPrefix + 1024 /*alignment*/;
  static_assert(kBytes <= 227 * 1024, "shared memory plan exceeds 227 KB");
  static constexpr int kSegBlocks = kKind == kHalf ? 16 : kKind == kSplit ? 4 : 1;   // k-blocks per segment
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

// One elected lane of a converged warp issues (the operands are the same in all lanes, so they can sit in uniform
// registers, which the instruction takes them from).
#define FUMA_MMA(group, kind)                                                                       \
  asm volatile(                                                                                     \
      "{\n\t.reg .pred p, q;\n\t"                                                                   \
      "elect.sync _|q, 0xffffffff;\n\t"                                                             \
      "setp.ne.b32 p, %4, 0;\n\t"                                                                   \
      "@q tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d), \
      "l"(a), "l"(b), "r"(idesc), "r"(acc)                                                          \
      : "memory")

template <bool kF8, bool kPair>
__device__ __forceinline__ void mma_issue(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (kPair) {
    if constexpr (kF8) FUMA_MMA("2", "f8f6f4");
    else FUMA_MMA("2", "f16");
  } else {
    if constexpr (kF8) FUMA_MMA("1", "f8f6f4");
    else FUMA_MMA("1", "f16");
  }
}

// Arrival of the issued MMAs' completion on `bar`; a pair: on the barrier at that offset in both CTAs. The lane is the one
// that issued the MMAs (the election of a full warp always gives the same).
template <bool kPair>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (kPair)
    asm volatile(
        "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}

__device__ __forceinline__ uint32_t in_cta0(const void* p) {   // the same shared-memory object in the pair's first CTA
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}

__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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

// This warp's lanes and `cols` columns of TMEM (rounded up to 16) times a factor per lane.
__device__ __forceinline__ void tmem_scale(uint32_t taddr, int cols, float s) {
#pragma unroll 1
  for (int c = 0; c < cols; c += 16) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr + c)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * s);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr + c)
        : "memory");
  }
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// (x: contiguous, y: rows, z: matrix); all planes. Issued by one elected lane of a converged warp. kPair: `bar` is a
// shared::cluster address, in either CTA of the pair.
template <bool kPair>
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if constexpr (kPair)
    asm volatile(
        "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, "
        "%4, %5}], [%6];\n\t}" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(0), "r"(bar)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];\n\t}" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(0), "r"(bar)
        : "memory");
}

// The same with the tile in one go: (64 columns, rows, chunks of 64 columns, matrix, plane), for widths that are whole chunks.
template <bool kPair>
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int y, int chunk, int z, uint32_t bar) {
  if constexpr (kPair)
    asm volatile(
        "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, "
        "%4, %5, %6}], [%7];\n\t}" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(y), "r"(chunk), "r"(z), "r"(0), "r"(bar)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], "
        "[%7];\n\t}" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(y), "r"(chunk), "r"(z), "r"(0), "r"(bar)
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

// Work units of a group: its tiles of kTileM rows (row maps), or the parts that its contraction is cut into (weight
// gradient: even parts of at most `cap` blocks of 128 rows; a group without rows has one, which writes zeros).
template <int kMode, int kTileM>
__device__ __forceinline__ int group_units(int64_t len, int cap) {
  const int n = (int)((len + kTileM - 1) / kTileM);
  if constexpr (kMode == kModeDw) return n ? (n + cap - 1) / cap : 1;
  else return n;
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

// One item's place: group, first A row, first column, k-blocks. Rows are this CTA's 128 of the tile.
struct Item {
  int kblocks;      // negative: no more items
  int g, n0;
  int nt;           // columns of the tile that exist, rounded up to what the MMA takes
  int row0;         // first A row (row maps) or first contraction row (weight gradient)
  int m0, rows;     // weight gradient: first output row; rows of the tile that exist (may be 0)
  int tail;         // weight gradient: contraction rows of the last k-block (0: all)
  int slot;         // kSplit: index of the tile's (weight gradient: the first segment's) row block among the scales
  int partial;      // weight gradient: 1 + the workspace matrix that takes the sum, or 0
  int pad[2];
};
constexpr int kRing = 4;

// The group that unit u falls into, and its units before u: a search over every p.span-th group's start, then a walk.
template <int kMode, int kTileM>
__device__ __forceinline__ int find_group(const GroupedArgs& p, const int* prefix, int u, int& c, int64_t& at, int64_t& len) {
  int lo = 0, hi = (p.G + p.span - 1) / p.span;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= u) lo = mid; else hi = mid;
  }
  int g = lo * p.span;
  c = u - prefix[lo];
  at = group_at(p.offsets, g, p.T);
  len = group_len(p.offsets, g, p.T);
  for (int n = group_units<kMode, kTileM>(len, p.cap); c >= n && g + 1 < p.G;) {
    c -= n;
    ++g;
    at = group_at(p.offsets, g, p.T);
    len = group_len(p.offsets, g, p.T);
    n = group_units<kMode, kTileM>(len, p.cap);
  }
  return g;
}

template <bool kPair>
__device__ __forceinline__ int tile_columns(const GroupedArgs& p, int n0) {
  constexpr int kStep = kPair ? 32 : 16;
  const int cols = p.N - n0;
  return cols < p.bn ? (cols + kStep - 1) / kStep * kStep : p.bn;
}

// Row maps: item -> tile.
template <int kBK, bool kPair>
__device__ __forceinline__ Item row_item(const GroupedArgs& p, const int* prefix, int item, int rank) {
  constexpr int kTileM = kPair ? 2 * kBM : kBM;
  Item t{};
  const int u = item / p.tiles_n;
  int c;
  int64_t at, len;
  t.g = find_group<kModeFwd, kTileM>(p, prefix, u, c, at, len);
  const int64_t r = (int64_t)c * kTileM + rank * kBM, left = len - r;
  t.row0 = (int)(at + r);
  t.rows = left < kBM ? (int)(left < 0 ? 0 : left) : kBM;
  t.n0 = (item - u * p.tiles_n) * p.bn;
  t.kblocks = (p.K + kBK - 1) / kBK;
  t.slot = (int)(at / kBM + t.g + r / kBM);
  t.nt = tile_columns<kPair>(p, t.n0);
  return t;
}

// Weight gradient: item -> a part of a group's contraction and an output tile, the tiles of a part one after the other, so
// that the CTAs work on the same rows at the same time and all but the first find them in L2. (One line of all tiles cut into
// equal stretches balances better and loses more to rows read again from HBM: 172 us against 141 at 120,000 rows.) Parts of
// cut groups go to the workspace, slot 2 * (first block) / cap + part: see grouped.cuh.
template <int kBK>
__device__ __forceinline__ Item wgrad_item(const GroupedArgs& p, const int* prefix, int item) {
  Item t{};
  const int tiles = p.tiles_m * p.tiles_n;
  const int u = item / tiles, tile = item - u * tiles;
  int c;
  int64_t at, len;
  t.g = find_group<kModeDw, kBM>(p, prefix, u, c, at, len);
  const int blocks = (int)((len + kBM - 1) / kBM), parts = blocks > p.cap ? (blocks + p.cap - 1) / p.cap : 1;
  const int each = (blocks + parts - 1) / parts;
  const int64_t r0 = (int64_t)c * each * kBM, r1 = r0 + (int64_t)each * kBM;
  const int n = r0 < len ? (int)((r1 < len ? r1 : len) - r0) : 0;
  t.row0 = (int)(at + r0);
  t.kblocks = (n + kBK - 1) / kBK;
  t.tail = n % kBK;
  t.m0 = (tile / p.tiles_n) * kBM;
  t.n0 = (tile % p.tiles_n) * p.bn;
  t.rows = p.M - t.m0 < kBM ? p.M - t.m0 : kBM;
  t.slot = (int)(at / kBM) + t.g + c * each;
  t.nt = tile_columns<false>(p, t.n0);
  if (parts > 1) t.partial = 1 + (int)(2 * (at / kBM) / p.cap) + c;
  return t;
}

template <int kKind, int kMode, bool kPair>
__global__ void __launch_bounds__(kGThreads, 1)
    grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                        const __grid_constant__ GroupedArgs p) {
  static_assert(!kPair || (kMode != kModeDw && kKind == kHalf),
                "the weight gradient clears rows of a stage, which a pair would share; pairs are for 16-bit operands");
  using L = GSmem<kKind, kPair>;
  constexpr int kP = L::kP, kBK = L::kBK;
  constexpr bool kScaled = kKind != kHalf;
  constexpr bool kAmn = kMode == kModeDw;                 // A contiguous along the tile
  constexpr bool kBmn = kMode != kModeFwd;
  constexpr int kTileM = kPair ? 2 * kBM : kBM;
  constexpr uint32_t kChunkMn = kP * kBK * 128;           // bytes between 64-element chunks (planes inside)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_c = smem + L::kStages * L::kStage;
  uint64_t* bar_full = reinterpret_cast<uint64_t*>(smem_c + L::kStaging);
  uint64_t* bar_empty = bar_full + L::kStages;
  uint64_t* bar_acc_full = bar_empty + L::kStages;   // [2]
  uint64_t* bar_acc_empty = bar_acc_full + 2;        // [2]
  uint64_t* bar_done = bar_acc_empty + 2;
  uint64_t* bar_clear = bar_done + 1;                // [kStages]
  uint64_t* bar_item_full = bar_clear + L::kStages;  // [kRing]
  uint64_t* bar_item_empty = bar_item_full + kRing;  // [kRing]
  Item* ring = reinterpret_cast<Item*>(bar_item_empty + kRing);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ring + kRing);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* scan = reinterpret_cast<int*>(tmem_slot + 2);   // [kGThreads / 32]
  static_assert((3 * L::kStages + 5 + 2 * kRing) * 8 + kRing * sizeof(Item) + (2 + kGThreads / 32) * 4 <= 640, "barrier area");
  int* prefix = reinterpret_cast<int*>(smem_c + L::kStaging + 640);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kPair ? (int)(blockIdx.x & 1) : 0;       // cluster shape (2, 1, 1)
  const int first_item = kPair ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int item_step = kPair ? (int)(gridDim.x >> 1) : (int)gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_empty[s], kMode == kModeDw ? 2 : 1);   // the MMAs' completion; the weight gradient's clearing warp
      mbar_init(&bar_clear[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bar_acc_full[b], 1);
      mbar_init(&bar_acc_empty[b], kEpiWarps * (kPair ? 2 : 1));   // one arrival per epilogue warp
    }
    for (int r = 0; r < kRing; ++r) {
      mbar_init(&bar_item_full[r], 1);
      // epilogue warps, producer, MMA thread (of a pair's first CTA), clearing warp (weight gradient)
      mbar_init(&bar_item_empty[r], kEpiWarps + 1 + (rank == 0 ? 1 : 0) + (kMode == kModeDw ? 1 : 0));
    }
    mbar_init(bar_done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (kPair) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(512u)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(512u)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  // prefix[i] = work units before group i * span: threads 0..255 take `span` groups each, then a scan
  {
    const int g0 = threadIdx.x * p.span, g1 = threadIdx.x < kCoarse ? min(p.G, g0 + p.span) : 0;
    int sum = 0;
    int bad = 0;
    for (int g = g0; g < g1; ++g) {
      if (p.offsets) {
        const int64_t a = p.offsets[g], b = p.offsets[g + 1];
        bad |= a < 0 || b < a || b > p.T;
      }
      sum += group_units<kMode, kTileM>(group_len(p.offsets, g, p.T), p.cap);
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
    if (threadIdx.x < kCoarse) prefix[threadIdx.x] = base;
    if (threadIdx.x == kCoarse) prefix[kCoarse] = base;   // threads from kCoarse on add nothing: the total
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncwarp();
  if constexpr (kPair) cluster_sync();
  else __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const int units = prefix[kCoarse];

  if (warp < kEpiWarp0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCtrlRegs));
    if (warp == 0) {
      // ---------------- producer (the whole warp runs the loop, one lane issues)
      const uint32_t smem0 = smem_u32(smem);
      const uint32_t full0 = __shfl_sync(kFull, kPair ? in_cta0(bar_full) : smem_u32(bar_full), 0);
      int it = 0;
      bool ok = true;
      for (int n = 0; ok; ++n) {
        ok = __all_sync(kFull, mbar_wait(&bar_item_full[n % kRing], (n / kRing) & 1, abort_flag, p.err, kErrWaitFull));
        if (!ok) break;
        const Item& t = ring[n % kRing];
        const int kblocks = __shfl_sync(kFull, t.kblocks, 0), g = __shfl_sync(kFull, t.g, 0);
        const int nt = __shfl_sync(kFull, t.nt, 0), n0 = __shfl_sync(kFull, t.n0, 0);
        const int row0 = __shfl_sync(kFull, t.row0, 0), m0 = kMode == kModeDw ? __shfl_sync(kFull, t.m0, 0) : 0;
        if (lane == 0) mbar_arrive(&bar_item_empty[n % kRing]);
        if (kblocks < 0) break;
        const int cols = kPair ? nt / 2 : nt;             // of B in this CTA
        const int nb = n0 + rank * cols;
        const int loads = !kBmn ? 1 : p.wide_b ? p.box_b / 64 : (cols + 63) / 64;   // chunks of B that arrive
        const uint32_t bytes = kP * (L::kA + loads * (kBmn ? kBK * 128 : p.box_b * L::kRowBytes)) * (kPair ? 2 : 1);
        for (int kt = 0; kt < kblocks; ++kt, ++it) {
          const int s = it % L::kStages;
          if (it >= L::kStages) {
            ok = __all_sync(kFull, mbar_wait(&bar_empty[s], ((it / L::kStages) - 1) & 1, abort_flag, p.err, kErrWaitEmpty));
            if (!ok) break;
          }
          const uint32_t a = smem0 + s * L::kStage, b = a + kP * L::kA, bar = full0 + s * 8;
          if (rank == 0 && lane == 0) mbar_expect_tx(&bar_full[s], bytes);
          __syncwarp();
          // (one load where the width allows: each takes the producer about 100 cycles, and a stage's MMAs 512)
          if constexpr (kAmn) {
            if (p.wide_a) {
              tma_load_5d<kPair>(a, &tmA, row0 + kt * kBK, m0 / 64, 0, bar);
            } else {
#pragma unroll
              for (int c = 0; c < kBM / 64; ++c)
                tma_load_4d<kPair>(a + c * kChunkMn, &tmA, m0 + c * 64, row0 + kt * kBK, 0, bar);
            }
          } else {
            tma_load_4d<kPair>(a, &tmA, kt * kBK, row0, 0, bar);
          }
          if constexpr (kBmn) {
            const int y = kMode == kModeDw ? row0 + kt * kBK : kt * kBK, z = kMode == kModeDw ? 0 : g;
            if (p.wide_b) {
              tma_load_5d<kPair>(b, &tmB, y, nb / 64, z, bar);
            } else {
#pragma unroll
              for (int c = 0; c < kMaxBN / 64; ++c)
                if (c < loads) tma_load_4d<kPair>(b + c * kChunkMn, &tmB, nb + c * 64, y, z, bar);
            }
          } else {
            tma_load_4d<kPair>(b, &tmB, kt * kBK, nb, g, bar);
          }
        }
      }
      if (*abort_flag && rank == 0 && lane == 0) {
        for (int j = it - 1; j >= 0 && j >= it - L::kStages; --j) {
          for (uint32_t i = 0; i < kWaitLimit && !mbar_try(&bar_full[j % L::kStages], (j / L::kStages) & 1); ++i) {
          }
        }
      }
      __syncwarp();
    } else if (warp == 1 && rank == 0) {
      // ---------------- MMA issue (the whole warp runs the loop, one lane issues)
      const uint32_t fmt = p.mma_format;   // operand format bits of the instruction descriptor
      const uint32_t idesc0 = (1u << 4) | (fmt << 7) | (fmt << 10) | (kAmn ? 1u << 15 : 0u) | (kBmn ? 1u << 16 : 0u) |
                              ((uint32_t)(kTileM >> 4) << 24);
      // descriptors of stage 0, first plane, first step; the rest is constants added to the address field (units of
      // 16 bytes; shared memory stays below its 14 bits)
      const uint32_t a0 = smem_u32(smem), b0 = a0 + kP * L::kA;
      // MN-major tiles: loaded chunk by chunk, a chunk's planes follow one another; in one go, a plane's chunks do
      const uint32_t chunk_a = p.wide_a ? kBK * 128 : kChunkMn, chunk_b = p.wide_b ? kBK * 128 : kChunkMn;
      const uint64_t da0 = kAmn ? smem_desc_mn128(a0, chunk_a) : L::kRowBytes == 64 ? smem_desc_k64(a0) : smem_desc_sw128(a0);
      const uint64_t db0 = kBmn ? smem_desc_mn128(b0, chunk_b) : L::kRowBytes == 64 ? smem_desc_k64(b0) : smem_desc_sw128(b0);
      constexpr uint32_t kStepA = (kAmn ? 2048 : 32) / 16, kStepB = (kBmn ? 2048 : 32) / 16;
      const uint32_t plane_a = (!kAmn ? L::kA : p.wide_a ? kBM / 64 * kBK * 128 : kBK * 128) / 16;
      const uint32_t plane_b = (!kBmn ? p.box_b * L::kRowBytes : p.wide_b ? p.box_b / 64 * (kBK * 128) : kBK * 128) / 16;
      constexpr int kSteps = kBK * L::kElem / 32;
      const uint32_t tm = __shfl_sync(kFull, tmem, 0);
      const uint32_t empty0 = smem_u32(bar_empty), accf0 = smem_u32(bar_acc_full);
      int s = 0, phase = 0, seg = 0;
      uint32_t clear_phase = 0;   // one bit per stage
      bool ok = true;
      bool ready = false;         // the next stage's barrier was seen complete already
      for (int n = 0; ok; ++n) {
        ok = __all_sync(kFull, mbar_wait(&bar_item_full[n % kRing], (n / kRing) & 1, abort_flag, p.err, kErrWaitFull));
        if (!ok) break;
        const int kblocks = __shfl_sync(kFull, ring[n % kRing].kblocks, 0), nt = __shfl_sync(kFull, ring[n % kRing].nt, 0);
        const int tail = kMode == kModeDw ? __shfl_sync(kFull, ring[n % kRing].tail, 0) : 0;
        if (lane == 0) mbar_arrive(&bar_item_empty[n % kRing]);
        if (kblocks < 0) break;
        const uint32_t idesc = idesc0 | ((uint32_t)(nt >> 3) << 17);
        for (int kt = 0; kt < kblocks; ++kt) {
          const int buf = seg & 1;
          const bool first = kt % L::kSegBlocks == 0;
          if (first && seg >= 2) {
            ok = __all_sync(kFull, mbar_wait(&bar_acc_empty[buf], ((seg >> 1) - 1) & 1, abort_flag, p.err, kErrWaitAccEmpty));
            if (!ok) break;
          }
          int steps = kSteps;
          if (kMode == kModeDw && kt == kblocks - 1 && tail) {
            // the last k-block of a group ends inside the tile: only whole steps of 16 rows run, and warp 2 has
            // cleared the rest of the last one
            steps = (tail + 15) / 16;
            ok = __all_sync(kFull, mbar_wait(&bar_clear[s], (clear_phase >> s) & 1, abort_flag, p.err, kErrWaitSplit));
            clear_phase ^= 1u << s;
          } else if (!ready) {
            ok = __all_sync(kFull, mbar_wait(&bar_full[s], phase, abort_flag, p.err, kErrWaitFull));
          }
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t da = da0 + (uint32_t)(s * (L::kStage / 16)), db = db0 + (uint32_t)(s * (L::kStage / 16));
          const uint32_t acc_d = tm + (uint32_t)(buf * kMaxBN);
          const uint32_t empty = empty0 + s * 8;
          if (++s == L::kStages) {
            s = 0;
            phase ^= 1;
          }
          // a look at the next stage's barrier, its latency behind this stage's MMAs
          const bool peek = mbar_test(&bar_full[s], phase);
#pragma unroll
          for (int kk = 0; kk < kSteps; ++kk) {
            if (kMode == kModeDw && kk >= steps) break;
            const uint32_t acc = (kk == 0 && first) ? 0u : 1u;
            const uint64_t dak = da + kk * kStepA, dbk = db + kk * kStepB;
            if constexpr (kKind == kSplit) {   // the small products first
              mma_issue<false, kPair>(acc_d, dak, dbk + plane_b, idesc, acc);
              mma_issue<false, kPair>(acc_d, dak + plane_a, dbk, idesc, 1u);
              mma_issue<false, kPair>(acc_d, dak, dbk, idesc, 1u);
            } else {
              mma_issue<kKind == kFp8, kPair>(acc_d, dak, dbk, idesc, acc);
            }
          }
          commit<kPair>(empty);
          if (kt % L::kSegBlocks == L::kSegBlocks - 1 || kt == kblocks - 1) {
            commit<kPair>(accf0 + buf * 8);
            ++seg;
          }
          ready = __all_sync(kFull, peek);
        }
      }
      __syncwarp();
      if constexpr (kPair)
        asm volatile(
            "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
            "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar_done))
            : "memory");
      else
        commit<false>(smem_u32(bar_done));
      for (uint32_t i = 0; i < kWaitLimit && !mbar_try(bar_done, 0); ++i) {
      }
      __syncwarp();
    } else if (kMode == kModeDw && warp == 2) {
      // ---------------- clearing: in the last k-block of a group, the rows behind its end belong to the next group and
      // must not count, whatever they hold; those of the last MMA step are cleared in both operands (0 x inf would be NaN)
      int it = 0;
      Item t;
      for (int n = 0;; ++n) {
        bool ok = mbar_wait(&bar_item_full[n % kRing], (n / kRing) & 1, abort_flag, p.err, kErrWaitFull);
        ok = __all_sync(kFull, ok);
        if (!ok) break;
        t = ring[n % kRing];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_item_empty[n % kRing]);
        if (t.kblocks < 0) break;
        // every stage's barrier in order, also where nothing is to clear, and no stage is loaded again before this warp has
        // seen it full: a wait by parity means nothing to a warp that is two phases behind
        for (int kt = 0; kt < t.kblocks; ++kt) {
          const int s = (it + kt) % L::kStages;
          ok = __all_sync(kFull, mbar_wait(&bar_full[s], ((it + kt) / L::kStages) & 1, abort_flag, p.err, kErrWaitFull));
          if (!ok) break;
          if (lane == 0 && (kt + 1 < t.kblocks || !t.tail)) mbar_arrive(&bar_empty[s]);
        }
        if (!ok) break;
        if (t.tail) {
          const int s = (it + t.kblocks - 1) % L::kStages;
          uint8_t* sa = smem + s * L::kStage;
          uint8_t* sb = sa + kP * L::kA;
          const int dead = (t.tail + 15) / 16 * 16 - t.tail;
          const int chunks = kBM / 64 * kP, chunks_b = (p.wide_b ? p.box_b / 64 : (t.nt + 63) / 64) * kP;
          for (int i = lane; i < (chunks + chunks_b) * dead * 8; i += 32) {
            const int c = i / (dead * 8), r = (i / 8) % dead, j = i % 8;
            uint8_t* base = c < chunks ? sa + c * (kBK * 128) : sb + (c - chunks) * (kBK * 128);
            *reinterpret_cast<uint4*>(base + (t.tail + r) * 128 + j * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&bar_clear[s]);
            mbar_arrive(&bar_empty[s]);
          }
        }
        it += t.kblocks;
      }
      __syncwarp();
    } else if (warp == 3) {
      // ---------------- items
      if (lane == 0) {
        auto publish = [&](int n, const Item& t) {
          if (n >= kRing && !mbar_wait(&bar_item_empty[n % kRing], ((n / kRing) - 1) & 1, abort_flag, p.err, kErrWaitEmpty))
            return false;
          ring[n % kRing] = t;
          mbar_arrive(&bar_item_full[n % kRing]);
          return t.kblocks >= 0;
        };
        const int items = units * (kMode == kModeDw ? p.tiles_m * p.tiles_n : p.tiles_n);
        auto make = [&](int item) {
          if constexpr (kMode == kModeDw) return wgrad_item<kBK>(p, prefix, item);
          else return row_item<kBK, kPair>(p, prefix, item, rank);
        };
        Item last{};
        last.kblocks = -1;
        int item = first_item;
        for (int n = 0; publish(n, item < items ? make(item) : last); ++n) item += item_step;
      }
      __syncwarp();
    }
  } else {
    // ---------------- epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
    const int q = warp & 3, half = (warp - kEpiWarp0) >> 2;
    uint8_t* stage = smem_c + (warp - kEpiWarp0) * 4096;
    if constexpr (kMode != kModeDw) {
      // rows before the first and behind the last group: zeros
      const int64_t head = group_at(p.offsets, 0, p.T), tail = group_at(p.offsets, p.G, p.T);
      const int esize = p.out_dtype == kDtypeF32 ? 4 : 2, unit = p.N % 8 ? esize : 16;
      const int64_t row_bytes = (int64_t)p.N * esize, units_row = row_bytes / unit;
      const int64_t dead = units || head == tail ? head + (p.T - tail) : 0, n = dead * units_row;
      for (int64_t i = (int64_t)blockIdx.x * (kEpiWarps * 32) + threadIdx.x - kEpiWarp0 * 32; i < n;
           i += (int64_t)gridDim.x * (kEpiWarps * 32)) {
        const int64_t r = i / units_row, row = r < head ? r : tail + (r - head);
        uint8_t* c = static_cast<uint8_t*>(p.C) + row * row_bytes + (i - r * units_row) * unit;
        if (unit == 16) *reinterpret_cast<uint4*>(c) = make_uint4(0u, 0u, 0u, 0u);
        else if (unit == 4) *reinterpret_cast<uint32_t*>(c) = 0u;
        else *reinterpret_cast<uint16_t*>(c) = 0u;
      }
    }
    const uint32_t acc_empty[2] = {kPair ? in_cta0(&bar_acc_empty[0]) : smem_u32(&bar_acc_empty[0]),
                                   kPair ? in_cta0(&bar_acc_empty[1]) : smem_u32(&bar_acc_empty[1])};
    const int hw = p.bn > 128 ? 128 : (p.bn + 63) / 64 * 32;   // columns of this warp: [half * hw, + hw)
    const int col0 = half * hw;
    int seg = 0;
    for (int n = 0;; ++n) {
      if (!__all_sync(kFull, mbar_wait(&bar_item_full[n % kRing], (n / kRing) & 1, abort_flag, p.err, kErrWaitFull))) break;
      const Item t = ring[n % kRing];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_item_empty[n % kRing]);
      if (t.kblocks < 0) break;
      if (kMode == kModeDw && t.kblocks == 0) {   // a group without rows: this item's share of its matrix, as one run
        const int esize = p.out_dtype == kDtypeF32 ? 4 : 2, unit = 16 / esize;
        const int64_t n = (int64_t)p.M * p.N, share = (n + p.tiles_m * p.tiles_n - 1) / (p.tiles_m * p.tiles_n);
        const int64_t i0 = min((t.m0 / kBM * p.tiles_n + t.n0 / p.bn) * share, n), i1 = min(i0 + share, n);
        const int64_t a = t.g * n + i0, b = t.g * n + i1;
        const int64_t lo = min((a + unit - 1) / unit * unit, b), hi = max(b / unit * unit, lo);   // 16-byte steps in [lo, hi)
        const int tid = threadIdx.x - kEpiWarp0 * 32;
        uint8_t* c = static_cast<uint8_t*>(p.C);
        for (int64_t i = lo + (int64_t)tid * unit; i < hi; i += (int64_t)kEpiWarps * 32 * unit)
          *reinterpret_cast<uint4*>(c + i * esize) = make_uint4(0u, 0u, 0u, 0u);
        const int64_t e = tid < unit ? a + tid : hi + (tid - unit);   // the ends, at most unit - 1 elements each
        if (tid < 2 * unit && e < (tid < unit ? lo : b)) {
          if (esize == 4) reinterpret_cast<float*>(c)[e] = 0.0f;
          else reinterpret_cast<uint16_t*>(c)[e] = 0;
        }
        continue;
      }
      const int segs = (t.kblocks + L::kSegBlocks - 1) / L::kSegBlocks;
      const int n0 = t.n0 + col0;
      const int rows = t.rows - q * 32;                        // of this warp (may be <= 0)
      const int ncols = rows <= 0 ? 0 : min(min(hw, p.bn - col0), p.N - n0);   // this warp's columns (may be <= 0)
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
      const float* sa = nullptr;
      const float* sb = nullptr;
      int64_t step_a = 0, step_b = 0;
      float a_next = 1.0f, b_next = 1.0f;
      if constexpr (kScaled) {
        // the scales are loaded one segment ahead, so that their latency hides behind the wait for its MMAs
        const int nblk = min(n0 / 128, p.blocks_n - 1);
        if constexpr (kKind == kFp8) {
          sa = p.scale_a + min((int64_t)t.row0 + q * 32 + lane, p.T - 1);
          step_a = p.T;
        } else if constexpr (kMode == kModeDw) {
          sa = p.scale_a + (t.m0 / 128) * p.scale_slots + t.slot;
          step_a = 1;
        } else {
          sa = p.scale_a + min((int64_t)t.slot, p.scale_slots - 1);
          step_a = p.scale_slots;
        }
        if constexpr (kMode == kModeDw) {
          sb = p.scale_b + nblk * p.scale_slots + t.slot;
          step_b = 1;
        } else if constexpr (kMode == kModeDx) {   // W's scales are [G][blocks of the contraction][blocks of the columns]
          sb = p.scale_b + (int64_t)t.g * segs * p.blocks_n + nblk;
          step_b = p.blocks_n;
        } else {
          sb = p.scale_b + ((int64_t)t.g * p.blocks_n + nblk) * segs;
          step_b = 1;
        }
        if (segs) {
          a_next = *sa;
          b_next = *sb;
        }
      }
      bool ok = true;
      for (int sg = 0; sg < segs; ++sg, ++seg) {
        const int buf = seg & 1;
        const float s_a = a_next, s_b = b_next;   // multiplied after the wait: the loads stay in flight
        if constexpr (kScaled) {
          const int nx = sg + 1 < segs ? sg + 1 : sg;
          a_next = sa[nx * step_a];
          b_next = sb[nx * step_b];
        }
        ok = mbar_wait(&bar_acc_full[buf], (seg >> 1) & 1, abort_flag, p.err, kErrWaitAcc);
        ok = __all_sync(kFull, ok && !*abort_flag);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        // the product of two scales may leave the fp32 range where the result does not (and 0 x inf is NaN): then it is applied as
        // two powers of two with half the exponent each. kSplit multiplies twice always, kFp8 takes the first factor to TMEM if a
        // row of the warp needs it (a multiplication more, or a branch to one, in its drain: 8 to 17 us of 186 a pass)
        float s = 1.0f, s2 = 1.0f;
        if constexpr (kKind == kFp8) s = s_a * s_b;
        const bool wide = kKind == kFp8 && __any_sync(kFull, s == 0.0f || s > 3.402823466e38f);
        if (kKind == kSplit || (wide && s == s)) {   // (a scale that is NaN makes the sums NaN)
          const int e = (int)(__float_as_uint(s_a) >> 23) + (int)(__float_as_uint(s_b) >> 23) - 254, h = e >> 1;
          s = __uint_as_float((uint32_t)(h + 127) << 23);
          s2 = __uint_as_float((uint32_t)(e - h + 127) << 23);
        }
        if (wide) tmem_scale(tmem + (uint32_t)(buf * kMaxBN + col0) + ((uint32_t)(q * 32) << 16), ncols, s2);
        const uint32_t taddr = tmem + (uint32_t)(buf * kMaxBN + col0) + ((uint32_t)(q * 32) << 16);
#pragma unroll
        for (int c = 0; c < 4; c += 2) {
          if (c * 32 < ncols) {   // two loads in flight; the second may read columns that nobody uses
            uint32_t r[2][32];
            tmem_ld32(taddr + c * 32, r[0]);
            tmem_ld32(taddr + c * 32 + 32, r[1]);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int u = 0; u < 32; ++u) {
                float& a = acc[(c + h) * 32 + u];
                const float v = __uint_as_float(r[h][u]);
                if constexpr (kKind == kFp8) a = fmaf(v, s, a);
                else if constexpr (kKind == kSplit) a = fmaf(v * s, s2, a);
                else a += v;
              }
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          if constexpr (kPair) arrive_cluster(acc_empty[buf]);
          else mbar_arrive(&bar_acc_empty[buf]);
        }
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
      // rows out: 128 bytes of each of the warp's 32 rows at a time through the staging area (16-byte
      // chunk j of row r at j ^ (r & 7)), so a store instruction writes 4 rows x 128 bytes. (TMA stores from the staging
      // area queue behind the producer's loads: the fp8 map took 128 us with them and 107 without.)
      const bool partial = kMode == kModeDw && t.partial;
      const int out_dtype = partial ? kDtypeF32 : p.out_dtype;
      const int64_t ld = partial ? p.ldw : p.N;
      const bool rows16 = kPair || partial || p.N % 8 == 0;   // output rows in 16-byte steps (pairs: always)
      const int64_t y0 = (kMode == kModeDw ? (int64_t)(partial ? t.partial - 1 : t.g) * p.M + t.m0 : t.row0) + q * 32;
      const int x0 = n0;
      uint8_t* out = static_cast<uint8_t*>(partial ? p.work : p.C);
      const int rr = lane >> 3, jj = lane & 7;
      if (out_dtype == kDtypeF32) {
        float* o = reinterpret_cast<float*>(out) + (y0 + rr) * ld + x0 + jj * 4;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c * 32 < ncols) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<float4*>(stage + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                  make_float4(acc[c * 32 + 4 * j], acc[c * 32 + 4 * j + 1], acc[c * 32 + 4 * j + 2], acc[c * 32 + 4 * j + 3]);
            __syncwarp();
            if (!rows16) {
              if (c * 32 + lane < ncols)
#pragma unroll 4
                for (int r = 0; r < min(rows, 32); ++r)
                  reinterpret_cast<float*>(out)[(y0 + r) * ld + x0 + c * 32 + lane] =
                      *reinterpret_cast<const float*>(stage + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
            } else if (c * 32 + jj * 4 < ncols) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int r = i * 4 + rr;
                const float4 v = *reinterpret_cast<const float4*>(stage + r * 128 + ((jj ^ (r & 7)) << 4));
                if (r < rows) *reinterpret_cast<float4*>(o + i * 4 * ld + c * 32) = v;
              }
            }
          }
        }
      } else {
        uint16_t* o = reinterpret_cast<uint16_t*>(out) + (y0 + rr) * ld + x0 + jj * 8;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (c * 64 < ncols) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float* a = acc + c * 64 + 8 * j;
              *reinterpret_cast<uint4*>(stage + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                  make_uint4(pack_half(a[0], a[1], out_dtype), pack_half(a[2], a[3], out_dtype),
                             pack_half(a[4], a[5], out_dtype), pack_half(a[6], a[7], out_dtype));
            }
            __syncwarp();
            if (!rows16) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int k = h * 32 + lane;
                uint16_t* col = reinterpret_cast<uint16_t*>(out) + y0 * ld + x0 + c * 64 + k;
                if (c * 64 + k < ncols)
#pragma unroll 4
                  for (int r = 0; r < min(rows, 32); ++r)
                    col[r * ld] =
                        *reinterpret_cast<const uint16_t*>(stage + r * 128 + (((k >> 3) ^ (r & 7)) << 4) + (k & 7) * 2);
              }
            } else if (c * 64 + jj * 8 < ncols) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int r = i * 4 + rr;
                const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + ((jj ^ (r & 7)) << 4));
                if (r < rows) *reinterpret_cast<uint4*>(o + i * 4 * ld + c * 64) = v;
              }
            }
          }
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncwarp();
  if constexpr (kPair) cluster_sync();   // neither CTA leaves while the other may still signal or read its shared memory
  else __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if constexpr (kPair)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ---- joining the chunks of the weight gradient --------------------------------------------------
// dW[g] = sum over the group's parts, in order, for groups that were cut. Block row y takes the y-th such
// group (there are fewer than T / 128 / cap of them), found by a count over all groups: 256 threads with a run each.
__global__ void __launch_bounds__(256) grouped_join_kernel(const __grid_constant__ GroupedArgs p) {
  __shared__ int count[8], found;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int per = (p.G + 255) / 256, g0 = threadIdx.x * per, g1 = min(p.G, g0 + per);
  const int64_t most = (int64_t)p.cap * kBM;
  int n = 0;
  for (int g = g0; g < g1; ++g) n += group_len(p.offsets, g, p.T) > most;
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
      if (group_len(p.offsets, g, p.T) > most && before++ == y) found = g;
  }
  __syncthreads();
  const int g = found;
  if (g < 0) return;
  const int64_t at = group_at(p.offsets, g, p.T), len = group_len(p.offsets, g, p.T);
  const int parts = group_units<kModeDw, kBM>(len, p.cap);
  const int w4 = p.ldw / 4;                  // the parts' rows are padded to 8 columns
  const int64_t n4 = (int64_t)p.M * w4;
  const float* work = static_cast<const float*>(p.work) + 2 * (at / kBM) / p.cap * n4 * 4;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n4; i += (int64_t)gridDim.x * blockDim.x) {
    float4 s = ld4_stream(work + i * 4);
#pragma unroll 4
    for (int c = 1; c < parts; ++c) s += ld4_stream(work + (c * n4 + i) * 4);
    if (p.ldw == p.N) {
      const int64_t o = ((int64_t)g * n4 + i) * 4;
      if (p.out_dtype == kDtypeF32)
        st4(static_cast<float*>(p.C) + o, s);
      else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.C) + o) =
            make_uint2(pack_half(s.x, s.y, p.out_dtype), pack_half(s.z, s.w, p.out_dtype));
    } else {
      const int64_t m = i / w4;
      const int n = (int)(i - m * w4) * 4;
      const int64_t o = ((int64_t)g * p.M + m) * p.N + n;
      const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (n + k >= p.N) break;
        if (p.out_dtype == kDtypeF32) static_cast<float*>(p.C)[o + k] = v[k];
        else static_cast<uint16_t*>(p.C)[o + k] = (uint16_t)(pack_half(v[k], 0.0f, p.out_dtype) & 0xffffu);
      }
    }
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
// 8 rows in flight each, and join in shared memory. Row blocks cut into more than 4 pieces (many small groups):
// a warp per piece, no joining. 20,000 rows of 512 bf16 in 2,000 groups: 9.2 us, sharing every piece 28; 50,021 rows of
// 392 in 301 groups: 15.7, a warp per piece 80. Bound by latency (120,000 rows of 640: 154 MB in 34 us); all of a block's
// rows in registers ahead of the offsets took 64.
// kVec: rows 16-byte aligned.
template <int kDtype, bool kVec>
__global__ void __launch_bounds__(256, kVec ? 4 : 2) grouped_colsum_kernel(const void* __restrict__ x, int64_t ld,
                                                             const int64_t* __restrict__ off, int G, int shared,
                                                             int64_t T, int N, float* __restrict__ part) {
  __shared__ float sm[8][256 + 8];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int n = blockIdx.y * 256 + lane * 8;
  const int groups = shared ? 1 : G;
  const int64_t b0 = (int64_t)blockIdx.x * kSumRows, b1 = min(T, b0 + kSumRows);
  // the groups of the block's rows: from the first that ends behind b0 to the first that ends behind b1 - 1, by counting
  // those that end before (independent loads; a binary search's dependent ones took longer than the sums of 128 rows)
  __shared__ int count[8];
  int n_end = 0;   // ends <= b0, and in the upper half ends < b1
  for (int g = threadIdx.x; g < groups; g += 256) {
    const int64_t end = sum_bound(off, g + 1, G, T, shared);
    n_end += (end <= b0) + ((end < b1) << 16);
  }
  n_end = __reduce_add_sync(kFull, n_end);
  if (lane == 0) count[w] = n_end;
  __syncthreads();
  n_end = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) n_end += count[i];
  const int g0 = n_end & 0xffff, g1 = min(groups, (n_end >> 16) + 1);
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
          if (r + i * step < r1) {
            if constexpr (kVec) raw[i].load(x, (r + i * step) * ld + n);
            else raw[i].load_some(x, (r + i * step) * ld + n, min(8, N - n));
          }
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
      if constexpr (kVec) {
        if (n < N) {
          st4(out + n, make_float4(s[0], s[1], s[2], s[3]));
          st4(out + n + 4, make_float4(s[4], s[5], s[6], s[7]));
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (n + k < N) out[n + k] = s[k];
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
#pragma unroll 8
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

// ---- fp32 -> two fp16 planes under block scales ------------------------------------------------------
// One thread block per 128 x 128 block: 8 columns of 8 rows per thread, all loaded before the largest magnitude is
// known, split and written: one pass, 4 bytes in and 4 out per value. 16-byte stores: 66 us where 4 columns of 16 rows
// took 79 (and 66 with registers for a third resident block, which spills). Row blocks: of the ragged rows, the
// 128-row tiles of each group (counted from the group's first row, as the maps cut it; the tile's slot is group
// start / 128 + group + tile, distinct because one tile or one group further on moves it by at least 1), or, with
// mat_rows > 0, of matrices of mat_rows rows each, but (given offsets) those of groups without rows. A value that is not
// finite keeps hi alone and does not set the scale.
// kVec: rows 16-byte aligned. Planes [rows][ldp], ldp = cols rounded up to 8.
template <bool kVec>
__global__ void __launch_bounds__(256) split_blocks_kernel(const float* __restrict__ x, int64_t ldx, int64_t rows,
                                                           int cols, const int64_t* __restrict__ off, int G,
                                                           int mat_rows, int64_t T, __half* __restrict__ out,
                                                           float* __restrict__ scales, int64_t slots) {
  __shared__ uint32_t wmax[8];
  const int kblocks = (cols + 127) / 128;
  const int64_t slot = blockIdx.x / kblocks;
  const int kb = (int)(blockIdx.x - slot * kblocks);
  int64_t row0, n, scale_at;
  if (mat_rows > 0) {
    const int blocks = (mat_rows + 127) / 128;
    const int64_t m = slot / blocks;
    if (off && group_len(off, (int)m, T) == 0) return;
    const int i = (int)(slot - m * blocks);
    row0 = m * mat_rows + i * 128;
    n = mat_rows - i * 128;
    scale_at = slot * kblocks + kb;
  } else {
    int lo = 0, hi = G;   // the last group with start / 128 + group <= slot
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (group_at(off, mid, rows) / 128 + mid <= slot) lo = mid; else hi = mid;
    }
    const int64_t at = group_at(off, lo, rows), i = slot - (at / 128 + lo);
    if (i < 0) return;
    row0 = at + i * 128;
    n = group_len(off, lo, rows) - i * 128;
    scale_at = kb * slots + slot;
  }
  if (n <= 0) return;
  if (n > 128) n = 128;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = kb * 128 + (lane & 15) * 8, r0 = w * 2 + (lane >> 4);
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 16 * i;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[i][k] = 0.0f;
    if (r < n) {
      const float* src = x + (row0 + r) * ldx + c;
      if constexpr (kVec) {
        if (c < cols) {
          const float4 a = ld4_stream(src), b = ld4_stream(src + 4);
          v[i][0] = a.x; v[i][1] = a.y; v[i][2] = a.z; v[i][3] = a.w;
          v[i][4] = b.x; v[i][5] = b.y; v[i][6] = b.z; v[i][7] = b.w;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (c + k < cols) v[i][k] = __ldcs(src + k);
      }
    }
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = __float_as_uint(v[i][j]) & 0x7fffffffu;
      m = max(m, b < 0x7f800000u ? b : 0u);
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(kFull, m, o));
  if (lane == 0) wmax[w] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, wmax[i]);
  int e = (int)(m >> 23) - 127 - 14;
  if (e < -126) e = -126;
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  if (threadIdx.x == 0) scales[scale_at] = __uint_as_float((uint32_t)(127 + e) << 23);
  const int ldp = (cols + 7) / 8 * 8;
  if (c >= ldp) return;
  const int64_t plane = rows * ldp;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 16 * i;
    if (r < n) {
      __half h[8], l[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float f = v[i][j] * inv;
        h[j] = __float2half_rn(f);
        l[j] = __float2half_rn(fabsf(f) <= 3.402823466e38f ? f - __half2float(h[j]) : 0.0f);
      }
      uint4 u;
      memcpy(&u, h, 16);
      *reinterpret_cast<uint4*>(out + (row0 + r) * ldp + c) = u;
      memcpy(&u, l, 16);
      *reinterpret_cast<uint4*>(out + plane + (row0 + r) * ldp + c) = u;
    }
  }
}

// ---- host side --------------------------------------------------------------------------------------

namespace {

template <int kKind, int kMode, bool kPair>
cudaError_t launch_grouped(const CUtensorMap (&m)[2], const GroupedArgs& p, int64_t max_items, cudaStream_t s) {
  using L = GSmem<kKind, kPair>;
  auto kern = grouped_gemm_kernel<kKind, kMode, kPair>;
  static thread_local uint64_t configured = 0;  // one bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(configured >> (dev & 63) & 1)) {
    cudaError_t st = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
    if (st != cudaSuccess) return st;
    configured |= uint64_t(1) << (dev & 63);
  }
  if constexpr (kPair) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(sm_count() / 2 * 2));
    cfg.blockDim = dim3(kGThreads);
    cfg.dynamicSmemBytes = L::kBytes;
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 2;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    // as many pairs as run at once: a pair that had to wait for another's end would start its share late
    static thread_local int resident[64];
    int& n = resident[dev & 63];
    if (n == 0 && (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1)) {
      (void)cudaGetLastError();
      n = sm_count() / 4;
    }
    cfg.gridDim = dim3((unsigned)(2 * (max_items < 1 ? 1 : max_items < n ? max_items : n)));
    return cudaLaunchKernelEx(&cfg, kern, m[0], m[1], p);
  } else {
    const int64_t sms = sm_count();
    const int grid = (int)(max_items < 1 ? 1 : max_items < sms ? max_items : sms);
    kern<<<grid, kGThreads, L::kBytes, s>>>(m[0], m[1], p);
    return cudaGetLastError();
  }
}

// Columns per tile: the whole width in even parts of at most 256, multiples of `step` (with block scales 256 or 128), and
// narrower tiles, down to 32, while there are no more of them than SMs: a call of a few rows is bound by how many SMs pull
// its matrices in, but a second round of tiles costs more than narrow tiles save. `tiles_rows` is what groups of any
// length have on average, half a tile more than their rows each. bf16: 24 rows,
// 768 -> 640, 8.1 us, at full width 9.3; 1,000 rows in 4 groups 9.1, at full width 10.3, 32 wide (two rounds) 11.7;
// 4,000 rows in 8 groups, 512 -> 512, 8.8, at full width 9.8.
int pick_bn(int N, int64_t tiles_rows, bool scaled, int step) {
  int bn;
  if (scaled) {
    bn = N > 128 ? 256 : 128;   // whole 128-blocks of the scales
  } else {
    const int parts = (N + kMaxBN - 1) / kMaxBN;
    bn = ((N + parts - 1) / parts + step - 1) / step * step;
  }
  for (;;) {
    const int half = scaled ? bn / 2 : (bn / 2 + 31) / 32 * 32;
    if (half < 32 || half == bn || tiles_rows * ((N + half - 1) / half) > sm_count()) break;
    bn = half;
  }
  return bn;
}

// CTA pairs (16-bit operands only): tiles of 256 rows, when the groups are long enough that the padding of their last tile
// (128 rows more on average) costs less than what a pair saves, and there are 8 tiles or more for every pair of SMs: with
// fewer, the last round's idle SMs cost what the pairs save. bf16, forward and input gradient: 120,000 rows in 16 groups,
// 640 -> 768 columns, 108 and 99 us, single CTAs 115 and 123; 32,768 rows in 32 groups, 512 -> 512 (4 tiles a pair), 26.7
// and 26.4 us, single 25.6 and 25.5. At 30,011 rows in 8 groups in fp32 pairs are slower (55.2 and 53.6 us, single 51.6
// and 50.9), and so they are in fp8 (184 us, 110): both have scales to fetch and sums to drain between the products,
// which a pair does in step.
bool use_pair(int64_t T, int G, int64_t items) { return T >= (int64_t)1024 * G && items >= (int64_t)4 * sm_count(); }

}  // namespace

int launch_grouped_rows(const GroupedOperands& o, GroupedArgs p, bool transposed, int* err, cudaStream_t s) {
  const bool fp8 = o.kind == kFp8, split = o.kind == kSplit;
  const int esize = fp8 ? 1 : 2, P = split ? 2 : 1;
  const int bk = fp8 ? 128 : split ? 32 : 64;
  const int64_t groups = p.G < p.T ? p.G : p.T;
  const int64_t tiles_rows = p.T / kBM + groups;   // upper bound: a partial tile per group
  p.bn = pick_bn(p.N, p.T / kBM + (groups + 1) / 2, fp8 || split, transposed ? 64 : 32);   // transposed: whole chunks of 64
  p.tiles_n = (p.N + p.bn - 1) / p.bn;
  p.tiles_m = 1;
  p.err = err;
  p.span = (p.G + kCoarse - 1) / kCoarse;
  p.mma_format = (!fp8 && !split && o.dtype == kDtypeBf16) ? 1u : 0u;
  const int64_t pair_items = (p.T / (2 * kBM) + groups) * p.tiles_n;
  const bool pair = o.kind == kHalf && p.N % 8 == 0 && p.bn > 128 && use_pair(p.T, p.G, pair_items);
  p.box_b = pair ? p.bn / 2 : p.bn;   // columns of the tile in this CTA: rows of W per load (forward)
  p.wide_b = transposed && p.N % (pair ? 128 : 64) == 0 && p.box_b % 64 == 0;
  p.wide_a = 0;
  const CUtensorMapDataType dt = fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                 : p.mma_format ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUtensorMapSwizzle ksw = split ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  CUtensorMap m[2];
  // A: [T rows, K], planes T * lda apart
  if (!make_map_4d(&m[0], dt, o.A, p.K, p.T, 1, P, o.lda * esize, p.T * o.lda * esize, p.T * o.lda * esize, bk, kBM, P,
                   ksw))
    return -1;
  // W: forward [G, N, K] with K contiguous along the contraction; input gradient [G, K, N] with the
  // output columns contiguous
  const int64_t brows = transposed ? p.K : p.N, bcols = transposed ? p.N : p.K;
  if (p.wide_b ? !make_map_5d(&m[1], dt, o.B, bcols, brows, p.G, P, o.ldb * 2, brows * o.ldb * 2, p.G * brows * o.ldb * 2,
                              bk, p.box_b / 64, P)
               : !make_map_4d(&m[1], dt, o.B, bcols, brows, p.G, P, o.ldb * esize, brows * o.ldb * esize,
                              p.G * brows * o.ldb * esize, transposed ? 64 : bk, transposed ? bk : p.box_b, P,
                              transposed ? CU_TENSOR_MAP_SWIZZLE_128B : ksw))
    return -1;
  const int64_t items = tiles_rows * p.tiles_n;
  cudaError_t st;
  if (pair)
    st = transposed ? launch_grouped<kHalf, kModeDx, true>(m, p, pair_items, s)
                    : launch_grouped<kHalf, kModeFwd, true>(m, p, pair_items, s);
  else if (fp8) st = launch_grouped<kFp8, kModeFwd, false>(m, p, items, s);
  else if (split)
    st = transposed ? launch_grouped<kSplit, kModeDx, false>(m, p, items, s)
                    : launch_grouped<kSplit, kModeFwd, false>(m, p, items, s);
  else
    st = transposed ? launch_grouped<kHalf, kModeDx, false>(m, p, items, s)
                    : launch_grouped<kHalf, kModeFwd, false>(m, p, items, s);
  return (int)st;
}

static int wgrad_bn(int N, bool split) {
  if (split) return N > 128 ? 256 : 128;   // whole 128-blocks of the scales
  const int parts = (N + kMaxBN - 1) / kMaxBN;
  return ((N + parts - 1) / parts + 63) / 64 * 64;
}

// Blocks of 128 rows per part of the weight gradient: long groups are cut so that the parts fill the SMs about twice
// over, but not below 16, where writing and joining the fp32 matrices costs as much as the products. At 120,000 rows in 16
// groups, 640 x 768: twice 134 + 17 us (products + joining), three times 140 + 22, four times 130 + 26.
static int wgrad_cap(int64_t T, int M, int N, bool split) {
  const int bn = wgrad_bn(N, split);
  const int64_t tiles = (int64_t)((M + kBM - 1) / kBM) * ((N + bn - 1) / bn);
  int64_t cap = T / kBM * tiles / ((int64_t)sm_count() * 2);
  if (cap < 16) cap = 16;
  return cap > (1 << 13) ? 1 << 13 : (int)cap;
}

int64_t grouped_wgrad_work_bytes(int64_t T, int M, int N, int dtype) {
  const int cap = wgrad_cap(T, M, N, dtype == kDtypeF32);
  if (T <= (int64_t)cap * kBM) return 0;
  return (2 * (T / kBM) / cap + 2) * (int64_t)M * ((N + 7) / 8 * 8) * 4;
}

int launch_grouped_wgrad(const GroupedOperands& o, GroupedArgs p, int* err, cudaStream_t s) {
  const bool split = o.kind == kSplit;
  const int P = split ? 2 : 1, bk = split ? 32 : 64;
  p.err = err;
  p.bn = wgrad_bn(p.N, split);
  p.tiles_n = (p.N + p.bn - 1) / p.bn;
  p.tiles_m = (p.M + kBM - 1) / kBM;
  p.span = (p.G + kCoarse - 1) / kCoarse;
  p.mma_format = (!split && o.dtype == kDtypeBf16) ? 1u : 0u;
  p.ldw = (p.N + 7) / 8 * 8;
  p.box_b = p.bn;
  p.wide_a = p.M % 64 == 0;
  p.wide_b = p.N % 64 == 0;
  p.cap = wgrad_cap(p.T, p.M, p.N, split);
  const CUtensorMapDataType dt = p.mma_format ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap m[2];
  auto operand = [&](CUtensorMap* map, const void* base, int cols, int64_t ld, bool wide, int chunks) {
    return wide ? make_map_5d(map, dt, base, cols, p.T, 1, P, ld * 2, p.T * ld * 2, p.T * ld * 2, bk, chunks, P)
                : make_map_4d(map, dt, base, cols, p.T, 1, P, ld * 2, p.T * ld * 2, p.T * ld * 2, 64, bk, P,
                              CU_TENSOR_MAP_SWIZZLE_128B);
  };
  if (!operand(&m[0], o.A, p.M, o.lda, p.wide_a, kBM / 64) || !operand(&m[1], o.B, p.N, o.ldb, p.wide_b, p.bn / 64))
    return -1;
  const int64_t items = (p.T / kBM / p.cap + p.G) * (int64_t)p.tiles_m * p.tiles_n;
  cudaError_t st = split ? launch_grouped<kSplit, kModeDw, false>(m, p, items, s)
                         : launch_grouped<kHalf, kModeDw, false>(m, p, items, s);
  if (st == cudaSuccess && p.T > (int64_t)p.cap * kBM) {
    const int64_t n4 = (int64_t)p.M * p.ldw / 4;
    int64_t bx = (n4 + 255) / 256;
    if (bx > 512) bx = 512;
    const int64_t long_groups = p.T / ((int64_t)p.cap * kBM);
    grouped_join_kernel<<<dim3((unsigned)bx, (unsigned)(long_groups < p.G ? long_groups : p.G)), 256, 0, s>>>(p);
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
    const bool vec = ld % 8 == 0 && N % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
    auto kern = dtype == kDtypeF32    ? (vec ? grouped_colsum_kernel<kDtypeF32, true> : grouped_colsum_kernel<kDtypeF32, false>)
                : dtype == kDtypeBf16 ? (vec ? grouped_colsum_kernel<kDtypeBf16, true> : grouped_colsum_kernel<kDtypeBf16, false>)
                                      : (vec ? grouped_colsum_kernel<kDtypeF16, true> : grouped_colsum_kernel<kDtypeF16, false>);
    kern<<<dim3((unsigned)((T + kSumRows - 1) / kSumRows), (unsigned)((N + 255) / 256)), 256, 0, s>>>(
        x, ld, off, G, shared, T, N, part);
    const cudaError_t st = cudaGetLastError();
    if (st != cudaSuccess) return st;
  }
  // few pieces per group: a warp joins a group's (2,000 groups of 10 rows: 8.5 us, a block per group 180; 16 groups of 7,500
  // rows the other way round: 5.4 us, a warp per group 8.1)
  const bool by_warp = groups >= 8 && T / groups < 8 * kSumRows;
  const int gy = by_warp ? (groups + kJoinWarps - 1) / kJoinWarps : groups;
  grouped_colsum_join_kernel<<<dim3((unsigned)((N + 31) / 32), (unsigned)gy), 32 * kJoinWarps, 0, s>>>(
      part, off, G, shared, T, N, out, dtype, by_warp);
  return cudaGetLastError();
}

int64_t split_slots(int64_t rows, int G) { return rows / 128 + G; }

void launch_split_blocks(const float* x, int64_t ldx, int64_t rows, int cols, const int64_t* off, int G, int mat_rows,
                         int64_t T, void* out, float* scales, cudaStream_t s) {
  const int64_t slots = mat_rows > 0 ? rows / mat_rows * ((mat_rows + 127) / 128) : split_slots(rows, G);
  const int64_t blocks = slots * ((cols + 127) / 128);
  const bool vec = ldx % 4 == 0 && cols % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  auto kern = vec ? split_blocks_kernel<true> : split_blocks_kernel<false>;
  kern<<<(unsigned)blocks, 256, 0, s>>>(x, ldx, rows, cols, off, G, mat_rows, T, static_cast<__half*>(out), scales, slots);
}

// 16-bit rows to a 16-byte pitch (for TMA): 8 values per lane in aligned 4-byte loads (a load covers a byte that is needed, so
// it stays in the allocation), as many lanes on a row as it has chunks. Columns behind the last hold nothing (the tensor maps
// end before them). Block column y is a matrix of mat_rows rows, left out if its group has no rows; without offsets, the
// one run of rows. Bound by HBM: 120,001
// rows of 641 and 767 values, 980 MB read and written, in 174 us.
__global__ void __launch_bounds__(256) pad_rows_kernel(const uint16_t* __restrict__ x, int64_t ldx, int64_t mat_rows, int cols,
                                                       uint16_t* __restrict__ out, int64_t ldo,
                                                       const int64_t* __restrict__ off, int64_t T, int lanes) {
  if (off && group_len(off, blockIdx.y, T) == 0) return;
  const int c8 = (cols + 7) / 8, per = 256 / lanes, l = threadIdx.x & (lanes - 1);
  const int64_t row0 = (int64_t)blockIdx.y * mat_rows;
  for (int64_t m = (int64_t)blockIdx.x * per + threadIdx.x / lanes; m < mat_rows; m += (int64_t)gridDim.x * per) {
    const uint16_t* src = x + (row0 + m) * ldx;
    uint4* dst = reinterpret_cast<uint4*>(out + (row0 + m) * ldo);
    const bool odd = reinterpret_cast<uintptr_t>(src) & 2;
    const uint32_t* words = reinterpret_cast<const uint32_t*>(src - odd);
#pragma unroll 4
    for (int j = l; j < c8; j += lanes) {
      uint32_t w[5];
#pragma unroll
      for (int k = 0; k < 5; ++k) w[k] = j * 8 + 2 * k < cols + odd ? __ldcs(words + j * 4 + k) : 0u;
      uint4 u;
      u.x = odd ? __funnelshift_r(w[0], w[1], 16) : w[0];
      u.y = odd ? __funnelshift_r(w[1], w[2], 16) : w[1];
      u.z = odd ? __funnelshift_r(w[2], w[3], 16) : w[2];
      u.w = odd ? __funnelshift_r(w[3], w[4], 16) : w[3];
      dst[j] = u;
    }
  }
}

void launch_pad_rows(const void* x, int64_t ldx, int64_t rows, int cols, void* out, int64_t ldo, const int64_t* off,
                     int mat_rows, int64_t T, cudaStream_t s) {
  int lanes = 1;
  while (lanes < 32 && lanes < (cols + 7) / 8) lanes *= 2;
  const int64_t m = off ? mat_rows : rows, mats = off ? rows / mat_rows : 1;
  const int64_t want = (m + 256 / lanes - 1) / (256 / lanes), most = (int64_t)8 * sm_count();
  pad_rows_kernel<<<dim3((unsigned)(want < most ? want : most), (unsigned)mats), 256, 0, s>>>(
      static_cast<const uint16_t*>(x), ldx, m, cols, static_cast<uint16_t*>(out), ldo, off, T, lanes);
}

}  // namespace fuma
