// Products of ragged groups of rows with a weight per group, and their
// gradients:
//
//   y_r = W_e x_r + b_e,   dx_r = W_e^T dy_r,   dW_e = sum_r dy_r x_r^T,
//   db_e = sum_r dy_r,     over the rows r of group e.
//
// The group sizes are known to the device only.  A launch has one block for
// every row tile that n rows in the given number of groups can fill at most;
// each block finds its group and rows from the offsets, and those past the
// last tile return.  Rows are read and written through `rows` where the
// groups' rows do not lie together, so no permuted copy is made.
//
// A block of four waves makes a tile of 128 output rows by 64 or 128 columns on
// the matrix cores, each wave half of both, from operands staged in LDS 64 or
// 128 bytes of the summed index at a time, the next stage's loads in flight while
// one is multiplied.  An operand whose summed index is innermost in memory
// ("along": rows of x, of W forward) is staged as it lies; one whose tile
// index is innermost ("across": W backward, both operands of dW) is staged as
// it lies too and transposed by the LDS reads.  The columns are the matrix
// cores' rows, so that a lane ends with four neighbouring columns of one output
// row.  Sums are float32.
//
// dW sums over rows: its blocks take a fixed number of rows of one group each.
// A group of one such part is stored at once; the others leave float32 parts,
// which a second kernel adds in row order.  Only those parts have a place in the
// workspace, so its size does not grow with the groups.
#include <algorithm>

#include "r2s_latent.h"

namespace r2s {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 128;      // output rows of a block's tile
constexpr int kWindow = 512;    // row numbers of a weights' gradient block in LDS, twice

using f32x4 = __attribute__((ext_vector_type(4))) float;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using i16x4 = __attribute__((ext_vector_type(4))) short;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using Lds = __attribute__((address_space(3))) char *;

// acc += A B over the 16 bytes per lane of the summed index (which elements
// they are does not matter, as long as both operands hold the same).
template <typename T>
__device__ __forceinline__ void multiply(u32x4 a, u32x4 b, f32x4 &acc) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], acc, 0, 0, 0);
  } else if constexpr (std::is_same<T, bf16_t>::value) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                  __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  } else {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                 __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
  }
}

// The groups' row ranges, safe for any offsets.
struct Groups {
  const int32_t *offsets;
  int64_t n;
  int32_t count;
  __device__ __forceinline__ int64_t bound(int64_t e) const {
    return min(max(static_cast<int64_t>(offsets[e]), int64_t{0}), n);
  }
};

// A group's parts that have a place in the workspace: all of several, but not an
// only one.
__device__ __forceinline__ uint32_t kept_parts(uint32_t parts) { return parts > 1u ? parts : 0u; }

// A part of a group: its rows [r0, r1), whether it is the group's only one, and
// else its place among the parts of all groups that have several.
struct Part {
  int32_t group;
  int64_t r0, r1;
  bool only;
  uint32_t place;
};

// Part `slot` of the groups cut into parts of `per` rows each.  With `rest` the
// rows past the last group follow as group `count`.  False past the last part.
// Called by whole waves.
__device__ __forceinline__ bool find_part(const Groups &g, bool rest, uint32_t per, uint32_t slot,
                                          Part &part) {
  uint32_t before = 0, kept_before = 0;
  const int32_t total = g.count + (rest ? 1 : 0);
  for (int32_t e0 = 0; e0 < total; e0 += 64) {
    const int32_t e = e0 + static_cast<int32_t>(lane_id());
    int64_t lo = 0, hi = 0;
    if (e < g.count)
      lo = g.bound(e), hi = g.bound(e + 1);
    else if (e < total)
      lo = g.bound(e), hi = g.n;
    const uint32_t parts = hi > lo ? static_cast<uint32_t>((hi - lo + per - 1) / per) : 0u;
    const uint32_t end = before + wave_inclusive_scan(parts);
    const uint32_t kept_end = kept_before + wave_inclusive_scan(kept_parts(parts));
    const uint64_t past = ballot(end > slot);
    if (past != 0) {
      const uint32_t src = static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(past))) - 1u;
      part.group = static_cast<int32_t>(readlane_u32(static_cast<uint32_t>(e), src));
      const uint32_t count = readlane_u32(parts, src), first = readlane_u32(end, src) - count;
      part.r0 = readlane_i64(lo, src) + static_cast<int64_t>(slot - first) * per;
      part.r1 = min(readlane_i64(hi, src), part.r0 + per);
      part.only = count == 1;
      part.place = readlane_u32(kept_end, src) - kept_parts(count) + (slot - first);
      return true;
    }
    before = readlane_u32(end, 63);
    kept_before = readlane_u32(kept_end, 63);
  }
  return false;
}

// ------------------------------------------------------------- staging ---

// The wave's loads to LDS have arrived, and so have the other waves': the next
// stage is in LDS, and the one that was multiplied last is free.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// An operand's stage is R x S bytes of LDS (S = 64 or 128 of the summed index) in
// 16-byte slots:
//   along   [R rows][S / 16 slots], slot s of row r at s ^ swizzle(r);
//   across  [S / sizeof(T) summed][R sizeof(T) / 16 slots], slot s of index c at
//           s ^ swizzle(c),
// so that the lanes that read together hit different ones of the 64 banks
// although LDS is filled in order by loads that go straight there.  The across
// order is made for tiles whose rows are in order (the weights' gradient).  Read
// in runs (the input's gradient) its lanes lie 16 columns apart and meet in
// banks, four at a time in tiles of 128 columns and two in those of 64.
// kRun: the tile's rows are taken kRun apart, four at a time (see Accumulator);
// 0: in order.
template <int S, int kRun>
__device__ __forceinline__ int along_swizzle(int r) {
  static_assert(kRun == 0 || S == 128, "runs of 128-byte rows");
  if constexpr (kRun > 0) return (r & 3) | ((r / kRun) & 1) << 2;
  return S == 128 ? r & 7 : (r >> 1) & 3;
}
template <typename T, int R>
__device__ __forceinline__ int across_swizzle(int c) {
  // f32: four runs of 64 bytes, 4 indices apart.  16 bits: eight runs of 32
  // bytes, indices c to c + 3 and c + 8 to c + 11; rows of 128 bytes put every
  // other index in the other half of the banks by themselves.
  if constexpr (sizeof(T) == 4)
    return ((c >> 2) & 3) << 2;
  else if constexpr (R == 128)
    return ((c & 3) | ((c >> 3) & 1) << 2) << 1;
  else
    return (((c >> 1) & 1) | ((c >> 3) & 1) << 1) << 1;
}

// The slots that a thread fills: q = i kThreads + threadIdx.x.
template <typename T, bool kAcross, int R, int S, int kRun = 0>
struct Slot {
  static constexpr int kSlots = S / 16;
  static constexpr int kCount = R * kSlots / kThreads;
  static constexpr int kPer = 16 / static_cast<int>(sizeof(T));  // elements
  int index;   // tile row (along) or summed index (across)
  int offset;  // elements from the stage's first, in the other direction
  __device__ __forceinline__ explicit Slot(int i) {
    const int q = i * kThreads + static_cast<int>(threadIdx.x);
    if constexpr (kAcross) {
      constexpr int kRow = R * static_cast<int>(sizeof(T)) / 16;
      index = q / kRow;
      offset = ((q % kRow) ^ across_swizzle<T, R>(index)) * kPer;
    } else {
      index = q / kSlots;
      offset = ((q % kSlots) ^ along_swizzle<S, kRun>(index)) * kPer;
    }
  }
};

// Fills slot i of the thread from 16 bytes at p.
__device__ __forceinline__ void load_slot(char *lds, int i, const void *p) {
  const int wave = static_cast<int>(wave_index());
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) void *)p,
      (__attribute__((address_space(3))) void *)(lds + (i * kThreads + wave * 64) * 16), 16, 0, 0);
}
// The same, or with zeros.
__device__ __forceinline__ void fill_slot(char *lds, int i, const void *p, bool some) {
  if (some) {
    load_slot(lds, i, p);
  } else {
    *reinterpret_cast<u32x4 *>(lds + (i * kThreads + threadIdx.x) * 16) = u32x4{0, 0, 0, 0};
  }
}
// 16 bytes at p of which the first `count` elements exist, zeros for the rest;
// p at any element.
template <typename T>
struct __attribute__((packed)) Unaligned {
  T v[16 / sizeof(T)];
};
template <typename T>
__device__ __forceinline__ u32x4 load_elements(const T *p, int64_t count) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  if (count >= kPer)
    return __builtin_bit_cast(u32x4, *reinterpret_cast<const Unaligned<T> *>(p));
  Pack<T, kPer> x;
#pragma unroll
  for (int j = 0; j < kPer; ++j) x.v[j] = j < count ? p[j] : static_cast<T>(0.0f);
  return __builtin_bit_cast(u32x4, x);
}
__device__ __forceinline__ void put_slot(char *lds, int i, u32x4 x) {
  *reinterpret_cast<u32x4 *>(lds + (i * kThreads + threadIdx.x) * 16) = x;
}

// Where this lane reads its 16 bytes of the summed index in a staged operand,
// for N tiles of 16 rows from `first` on: row n 16 + i of lane i (mod 16), or
// with kRun = 4 N row (i / 4) kRun + 4 n + i % 4.
template <typename T, bool kAcross, int R, int S, int N, int kRun = 0>
struct Fragments {
  static_assert(kRun == 0 || kRun == 4 * N, "a run per four lanes");
  static constexpr int kHalves = S / 64;  // what one matrix instruction (f32: four) sums over
  // along: one place per half; the tiles lie 16 (or 4) rows apart, which no
  // swizzle notices.  across: one place per tile; the halves lie half a slab
  // apart.
  int at[kAcross ? N : kHalves];
  __device__ __forceinline__ explicit Fragments(int first) {
    const int lane = static_cast<int>(lane_id()), i = lane % 16, q = lane / 16;
    if constexpr (!kAcross) {
      const int r = first + (kRun > 0 ? i / 4 * kRun + i % 4 : i);
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
        at[h] = r * S + ((h * 4 + q) ^ along_swizzle<S, kRun>(r)) * 16;
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if constexpr (sizeof(T) == 2) {
          // Sixteen lanes read 4 summed indices of 4 times 4 neighbours, 8
          // bytes each, and get 4 indices of one row each.
          const int c = q * 8 + i / 4;
          const int r = first + (kRun > 0 ? i % 4 * kRun + n * 4 : n * 16 + i % 4 * 4);
          at[n] = c * (R * 2) + ((r / 8) ^ across_swizzle<T, R>(c)) * 16 + r / 4 % 2 * 8;
        } else {
          const int c = q * 4;
          const int r = first + (kRun > 0 ? i / 4 * kRun + n * 4 + i % 4 : n * 16 + i);
          at[n] = c * (R * 4) + ((r / 4) ^ across_swizzle<T, R>(c)) * 16 + r % 4 * 4;
        }
      }
    }
  }
  __device__ __forceinline__ u32x4 load(const char *lds, int n, int half) const {
    if constexpr (!kAcross) {
      return *reinterpret_cast<const u32x4 *>(lds + at[half] + n * ((kRun > 0 ? 4 : 16) * S));
    } else if constexpr (sizeof(T) == 2) {
      const char *p = lds + at[n] + half * (32 * R * 2);
      const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) i16x4 *)p);
      const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) i16x4 *)(p + 4 * R * 2));
      u32x4 out;
      __builtin_memcpy(&out, &x, 8);
      __builtin_memcpy(reinterpret_cast<char *>(&out) + 8, &y, 8);
      return out;
    } else {
      const char *p = lds + at[n] + half * (16 * R * 4);
      u32x4 out;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        out[j] = *reinterpret_cast<const uint32_t *>(p + j * R * 4);
      return out;
    }
  }
};

// A wave's part of the tile: 64 rows by kCols / 2 columns, as tiles of 16 x 16
// of which a lane has four neighbouring columns of one row.  With kRuns its
// tiles' columns are neighbours too, kRun in all, so that it stores them by 16
// bytes: 500k x 64 x 64 bf16 forward 35 us, and 40 us with 8 bytes per tile.
template <int kCols, bool kRuns>
struct Accumulator {
  static constexpr int kA = kCols / 32, kB = kRows / 32, kRun = kRuns ? 4 * kA : 0;
  f32x4 v[kA][kB];
  __device__ __forceinline__ Accumulator() {
#pragma unroll
    for (int a = 0; a < kA; ++a)
#pragma unroll
      for (int b = 0; b < kB; ++b) v[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  static __device__ __forceinline__ int first_col() {
    return static_cast<int>(wave_index()) % 2 * (kCols / 2);
  }
  static __device__ __forceinline__ int first_row() {
    return static_cast<int>(wave_index()) / 2 * (kRows / 2);
  }
  // The tile's row, and the first of its four columns, that a lane has in v[a][b].
  static __device__ __forceinline__ int row(int b) {
    return first_row() + b * 16 + static_cast<int>(lane_id()) % 16;
  }
  static __device__ __forceinline__ int column(int a) {
    const int q = static_cast<int>(lane_id()) / 16;
    return first_col() + (kRuns ? q * kRun + a * 4 : a * 16 + q * 4);
  }
};

// acc += the products of a stage at `lds` (columns, then rows); kSums: sums +=
// the summed index's total of the row operand's rows, per lane its share.
template <typename T, bool kSums, int kColBytes, typename Acc, typename ColFragments,
          typename RowFragments>
__device__ __forceinline__ void multiply_stage(const char *lds, const ColFragments &cols,
                                               const RowFragments &rows, Acc &acc,
                                               float (&sums)[Acc::kB]) {
#pragma unroll
  for (int h = 0; h < ColFragments::kHalves; ++h) {
    u32x4 a[Acc::kA], b[Acc::kB];
#pragma unroll
    for (int i = 0; i < Acc::kA; ++i) a[i] = cols.load(lds, i, h);
#pragma unroll
    for (int i = 0; i < Acc::kB; ++i) b[i] = rows.load(lds + kColBytes, i, h);
#pragma unroll
    for (int i = 0; i < Acc::kA; ++i)
#pragma unroll
      for (int j = 0; j < Acc::kB; ++j) multiply<T>(a[i], b[j], acc.v[i][j]);
    if constexpr (kSums) {
#pragma unroll
      for (int j = 0; j < Acc::kB; ++j) {
        const Pack<T, 16 / sizeof(T)> x = __builtin_bit_cast(Pack<T, 16 / sizeof(T)>, b[j]);
#pragma unroll
        for (int k = 0; k < static_cast<int>(16 / sizeof(T)); ++k)
          sums[j] += static_cast<float>(x.v[k]);
      }
    }
  }
}

// The product over `steps` stages, two of them in LDS (one where there is but
// one).  stage(lds, step), the steps in order, puts a stage on its way to LDS,
// or reads it for commit(lds) to write it there.  More stages ahead measured
// slower: 16k x 1024 x 1024 bf16 forward and backward 254 us (229 now) with two of
// 64 bytes, 281 with three, 340 with four; blocks that share a CU hide more than
// depth.
template <int kStageBytes, typename Stage, typename Commit, typename Multiply>
__device__ __forceinline__ void pipeline(char *lds, int steps, Stage stage, Commit commit,
                                         Multiply multiply) {
  char *now = lds, *next = lds + kStageBytes;
  stage(now, 0);
  commit(now);
  for (int i = 0; i < steps; ++i) {
    stage_barrier();
    const bool more = i + 1 < steps;
    if (more) stage(next, i + 1);
    multiply(now);
    if (more) commit(next);
    char *t = now;
    now = next;
    next = t;
  }
}

// N neighbouring columns of an output row of `width`, at any element.
template <typename T, int N>
struct __attribute__((packed)) UnalignedRun {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ void store_run(T *row, int64_t col, int64_t width,
                                          const f32x4 (&v)[N / 4]) {
  if (col + N <= width) {
    constexpr int kMost = 16 / static_cast<int>(sizeof(T)), kStore = N < kMost ? N : kMost;
#pragma unroll
    for (int i = 0; i < N; i += kStore) {
      UnalignedRun<T, kStore> x;
#pragma unroll
      for (int j = 0; j < kStore; ++j) x.v[j] = static_cast<T>(v[(i + j) / 4][(i + j) % 4]);
      *reinterpret_cast<UnalignedRun<T, kStore> *>(row + col + i) = x;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (col + j < width) row[col + j] = static_cast<T>(v[j / 4][j % 4]);
  }
}

// ------------------------------------------------------------- kernels ---

// Rows times weights: out[r][j] = sum_c in[r][c] w(c, j), the forward
// (weight [m, k], summed over k) or with kBack the input's gradient (summed
// over m).  Blocks of one row tile are neighbours, and neighbours share an XCD:
// they read the same rows and weight.
//
// 16k x 1024 x 1024 bf16 in 16 groups: 66 us forward (520 TFLOP/s; 930 for one
// library product of these sizes), 69 us back (6.7e6 cycles of bank conflicts on
// 1.7e6 LDS instructions; none forward), bound by a stage's wait, by its LDS
// reads, which take as long as its products, and by 1160 blocks, of which the
// last run alone; at 32k x 2048 x 2048, 790 TFLOP/s.  500k x 64 x 64 bf16: 35 us
// forward, 128 MB at 3.7 TB/s, bound by the writes.  50k x 45 x 11 f32: 13 us,
// bound by the launch and a block's chain of offsets, rows, tile, store.
template <typename T, bool kBack, bool kVec, int kCols, int S>
__global__ __launch_bounds__(kThreads, kCols == 64 ? (kVec ? 4 : 3) : 2) void rows_kernel(
    const T *__restrict__ in, int64_t stride, const T *__restrict__ weight,
    const T *__restrict__ bias, Groups g, const int32_t *__restrict__ rows, int64_t k, int64_t m,
    uint32_t col_tiles, T *__restrict__ out) {
  extern __shared__ __attribute__((aligned(16))) char s_stage[];  // [1 or 2][cols, rows]
  __shared__ int32_t s_row[kRows];
  constexpr int kSlab = S / static_cast<int>(sizeof(T));
  constexpr int kColBytes = kCols * S, kStage = (kCols + kRows) * S;
  using Acc = Accumulator<kCols, true>;
  using RowSlot = Slot<T, false, kRows, S>;
  using ColSlot = Slot<T, kBack, kCols, S, kBack ? 0 : Acc::kRun>;
  const int64_t inner = kBack ? m : k, outer = kBack ? k : m;
  const uint32_t id = xcd_swizzle(blockIdx.x, gridDim.x);
  const int64_t j0 = static_cast<int64_t>(id % col_tiles) * kCols;
  Part part;
  if (!find_part(g, true, kRows, id / col_tiles, part)) return;
  const int32_t e = part.group;
  const int64_t r0 = part.r0, r1 = part.r1;
  if (threadIdx.x < kRows) {
    const int64_t i = r0 + threadIdx.x;
    int64_t r = -1;
    if (i < r1) {
      r = rows != nullptr ? rows[i] : i;
      if (r < 0 || r >= g.n) r = -1;
    }
    s_row[threadIdx.x] = static_cast<int32_t>(r);
  }
  __syncthreads();
  Acc acc;
  if (e < g.count && inner > 0) {
    const T *w = weight + static_cast<int64_t>(e) * m * k;
    // Addresses of the thread's slots in the next stage.  Rows and columns past
    // the tile's are some others: nothing of theirs is stored.
    const T *row_at[RowSlot::kCount], *col_at[ColSlot::kCount];
#pragma unroll
    for (int i = 0; i < RowSlot::kCount; ++i) {
      const RowSlot s(i);
      row_at[i] = in + static_cast<int64_t>(max(s_row[s.index], 0)) * stride + s.offset;
    }
#pragma unroll
    for (int i = 0; i < ColSlot::kCount; ++i) {
      const ColSlot s(i);
      if constexpr (kBack)
        col_at[i] = w + s.index * k + (j0 + s.offset < k ? j0 + s.offset : 0);
      else
        col_at[i] = w + min(j0 + s.index, m - 1) * k + s.offset;
    }
    const int64_t col_step = kBack ? kSlab * k : kSlab;
    u32x4 col_held[kVec ? 1 : ColSlot::kCount], row_held[kVec ? 1 : RowSlot::kCount];
    auto stage = [&](char *lds, int step) {
      const int64_t c0 = static_cast<int64_t>(step) * kSlab;
      if constexpr (!kVec) {
#pragma unroll
        for (int i = 0; i < ColSlot::kCount; ++i) {
          const ColSlot s(i);
          const int64_t count = !kBack             ? k - (c0 + s.offset)
                                : c0 + s.index < m ? k - (j0 + s.offset)
                                                   : 0;
          col_held[i] = load_elements<T>(col_at[i], count);
        }
#pragma unroll
        for (int i = 0; i < RowSlot::kCount; ++i)
          row_held[i] = load_elements<T>(row_at[i], inner - (c0 + RowSlot(i).offset));
      } else if (c0 + kSlab <= inner) {
#pragma unroll
        for (int i = 0; i < ColSlot::kCount; ++i) load_slot(lds, i, col_at[i]);
#pragma unroll
        for (int i = 0; i < RowSlot::kCount; ++i) load_slot(lds + kColBytes, i, row_at[i]);
      } else {
#pragma unroll
        for (int i = 0; i < ColSlot::kCount; ++i) {
          const ColSlot s(i);
          fill_slot(lds, i, col_at[i], c0 + (kBack ? s.index : s.offset) < inner);
        }
#pragma unroll
        for (int i = 0; i < RowSlot::kCount; ++i)
          fill_slot(lds + kColBytes, i, row_at[i], c0 + RowSlot(i).offset < inner);
      }
#pragma unroll
      for (int i = 0; i < ColSlot::kCount; ++i) col_at[i] += col_step;
#pragma unroll
      for (int i = 0; i < RowSlot::kCount; ++i) row_at[i] += kSlab;
    };
    auto commit = [&](char *lds) {
      if constexpr (!kVec) {
#pragma unroll
        for (int i = 0; i < ColSlot::kCount; ++i) put_slot(lds, i, col_held[i]);
#pragma unroll
        for (int i = 0; i < RowSlot::kCount; ++i) put_slot(lds + kColBytes, i, row_held[i]);
      }
    };
    const Fragments<T, kBack, kCols, S, Acc::kA, Acc::kRun> col_fragments(acc.first_col());
    const Fragments<T, false, kRows, S, Acc::kB> row_fragments(acc.first_row());
    float none[Acc::kB];
    pipeline<kStage>(
        s_stage, static_cast<int>((inner + kSlab - 1) / kSlab), stage, commit,
        [&](const char *lds) {
          multiply_stage<T, false, kColBytes>(lds, col_fragments, row_fragments, acc, none);
        });
  }
  // The biases of the lane's columns.
  f32x4 add[Acc::kA] = {};
  if (!kBack && bias != nullptr && e < g.count) {
    const T *b = bias + static_cast<int64_t>(e) * m;
#pragma unroll
    for (int a = 0; a < Acc::kA; ++a)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        add[a][i] = static_cast<float>(b[min(j0 + acc.column(a) + i, m - 1)]);
  }
#pragma unroll
  for (int b = 0; b < Acc::kB; ++b) {
    const int64_t at = s_row[acc.row(b)];
    if (at < 0) continue;
    f32x4 run[Acc::kA];
#pragma unroll
    for (int a = 0; a < Acc::kA; ++a) run[a] = acc.v[a][b] + add[a];
    store_run<T, Acc::kRun>(out + at * outer, j0 + acc.column(0), outer, run);
  }
}

// dW[m0 + row][k0 + col] (and db) of one part: `per` rows of one group.  The
// group's only part goes to v_weight and v_bias, others to their place in parts
// [places][m][k] and bias_parts [places][m].
//
// 16k x 1024 x 1024 bf16: 95 us, 360 TFLOP/s; both operands are read across, at
// half the LDS rate of operands read along, and a group of 4096 rows leaves 20 MB
// of parts.  Parts of equal length within a group were no faster (99 us).
// 500k x 64 x 64 bf16: 33 us, 128 MB read at 3.9 TB/s.
template <typename T, bool kVec, int kCols, int S>
__global__ __launch_bounds__(kThreads, kCols == 64 && kVec ? 3 : 2) void weights_kernel(
    const T *__restrict__ x, int64_t x_stride, const T *__restrict__ v_y, int64_t v_stride,
    Groups g, const int32_t *__restrict__ rows, int64_t k, int64_t m, uint32_t per,
    uint32_t m_tiles, uint32_t k_tiles, uint32_t places, float *__restrict__ parts,
    float *__restrict__ bias_parts, T *__restrict__ v_weight, T *__restrict__ v_bias) {
  extern __shared__ __attribute__((aligned(16))) char s_stage[];  // [2][cols, rows]
  // The rows' numbers, two windows by turns.
  __shared__ __attribute__((aligned(16))) int32_t s_row[2][kWindow];
  constexpr int kSlab = S / static_cast<int>(sizeof(T));
  constexpr int kColBytes = kCols * S, kStage = (kCols + kRows) * S;
  static_assert(kWindow % kSlab == 0 && kWindow % kThreads == 0, "whole slabs and waves");
  using Acc = Accumulator<kCols, false>;
  using RowSlot = Slot<T, true, kRows, S>;
  using ColSlot = Slot<T, true, kCols, S>;
  const uint32_t id = xcd_swizzle(blockIdx.x, gridDim.x), tiles = m_tiles * k_tiles;
  const uint32_t slot = id / tiles, tile = id - slot * tiles;
  const int64_t m0 = static_cast<int64_t>(tile / k_tiles) * kRows;
  const int64_t k0 = static_cast<int64_t>(tile % k_tiles) * kCols;
  Part part;
  if (!find_part(g, false, per, slot, part)) return;
  // Offsets that do not ascend could name more parts than there are places.
  if (!part.only && part.place >= places) return;
  const int32_t e = part.group;
  const int64_t r0 = part.r0, r1 = part.r1;
  const bool only = part.only;
  const int count = static_cast<int>(r1 - r0);
  // Window w's numbers on their way to LDS; past the part's end the last one's.
  auto fetch_rows = [&](int w) {
    if (rows == nullptr || w * kWindow >= count) return;
#pragma unroll
    for (int i = 0; i < kWindow / kThreads; ++i) {
      const int at = i * kThreads + static_cast<int>(wave_index()) * 64;
      const int32_t *p =
          rows + r0 + min(w * kWindow + at + static_cast<int>(lane_id()), count - 1);
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void *)p,
          (__attribute__((address_space(3))) void *)(s_row[w & 1] + at), 4, 0, 0);
    }
  };
  fetch_rows(0);
  stage_barrier();
  Acc acc;
  float sums[Acc::kB] = {};
  const bool with_bias = v_bias != nullptr && k0 == 0 && Acc::first_col() == 0;
  // The row of the part's place c < count.
  auto row_of = [&](int c) -> int64_t {
    if (rows == nullptr) return r0 + c;
    return min(max(static_cast<int64_t>(s_row[c / kWindow & 1][c % kWindow]), int64_t{0}),
               g.n - 1);
  };
  u32x4 col_held[kVec ? 1 : ColSlot::kCount], row_held[kVec ? 1 : RowSlot::kCount];
  auto stage = [&](char *lds, int step) {
    const int c0 = step * kSlab;
    // The next window, kWindow / kSlab steps before its first use.
    if (c0 % kWindow == 0) fetch_rows(c0 / kWindow + 1);
    const bool full = c0 + kSlab <= count;
#pragma unroll
    for (int i = 0; i < ColSlot::kCount; ++i) {
      const ColSlot s(i);
      const int64_t c = k0 + s.offset;
      const int at = full ? c0 + s.index : min(c0 + s.index, count - 1);
      const bool some = full || c0 + s.index < count;
      const T *p = x + row_of(at) * x_stride;
      if constexpr (!kVec)
        col_held[i] = load_elements<T>(p + c, some ? k - c : 0);
      else if (full)
        load_slot(lds, i, p + (c < k ? c : 0));
      else
        fill_slot(lds, i, p + (c < k ? c : 0), some);
    }
#pragma unroll
    for (int i = 0; i < RowSlot::kCount; ++i) {
      const RowSlot s(i);
      const int64_t c = m0 + s.offset;
      const int at = full ? c0 + s.index : min(c0 + s.index, count - 1);
      const bool some = full || c0 + s.index < count;
      const T *p = v_y + row_of(at) * v_stride;
      if constexpr (!kVec)
        row_held[i] = load_elements<T>(p + c, some ? m - c : 0);
      else if (full)
        load_slot(lds + kColBytes, i, p + (c < m ? c : 0));
      else
        fill_slot(lds + kColBytes, i, p + (c < m ? c : 0), some);
    }
  };
  auto commit = [&](char *lds) {
    if constexpr (!kVec) {
#pragma unroll
      for (int i = 0; i < ColSlot::kCount; ++i) put_slot(lds, i, col_held[i]);
#pragma unroll
      for (int i = 0; i < RowSlot::kCount; ++i) put_slot(lds + kColBytes, i, row_held[i]);
    }
  };
  const Fragments<T, true, kCols, S, Acc::kA> col_fragments(acc.first_col());
  const Fragments<T, true, kRows, S, Acc::kB> row_fragments(acc.first_row());
  const int steps = (count + kSlab - 1) / kSlab;
  if (with_bias)
    pipeline<kStage>(s_stage, steps, stage, commit, [&](const char *lds) {
      multiply_stage<T, true, kColBytes>(lds, col_fragments, row_fragments, acc, sums);
    });
  else
    pipeline<kStage>(s_stage, steps, stage, commit, [&](const char *lds) {
      multiply_stage<T, false, kColBytes>(lds, col_fragments, row_fragments, acc, sums);
    });
  if (v_weight != nullptr) {
    float *p = parts + static_cast<int64_t>(part.place) * m * k;
    T *w = v_weight + static_cast<int64_t>(e) * m * k;
#pragma unroll
    for (int b = 0; b < Acc::kB; ++b) {
      const int64_t r = m0 + acc.row(b);
      if (r >= m) continue;
#pragma unroll
      for (int a = 0; a < Acc::kA; ++a) {
        const int64_t c = k0 + acc.column(a);
        if (only)
          store_run<T, 4>(w + r * k, c, k, {acc.v[a][b]});
        else
          store_run<float, 4>(p + r * k, c, k, {acc.v[a][b]});
      }
    }
  }
  if (with_bias) {
    const int lane = static_cast<int>(lane_id());
#pragma unroll
    for (int j = 0; j < Acc::kB; ++j) {
      // The four lanes of a row hold the slab's quarters.
      float sum = sums[j];
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      const int64_t r = m0 + Acc::first_row() + j * 16 + lane % 16;
      if (lane < 16 && r < m) {
        if (only)
          v_bias[static_cast<int64_t>(e) * m + r] = static_cast<T>(sum);
        else
          bias_parts[static_cast<int64_t>(part.place) * m + r] = sum;
      }
    }
  }
}

// The weights' (blocks below weight_blocks) and biases' gradient of the groups
// that have no part or more than one: zeros, or the parts' sum, in row order.
// Many parts of small weights: kShare threads per element each add every
// kShare-th part and meet in LDS.  Few parts of large ones (kShare 1): a thread
// adds kRun neighbouring elements, 16 bytes of each part at a time.  16k x 1024
// x 1024 bf16: 12.6 us, and 20 us element by element.
template <typename T, int kShare>
__global__ __launch_bounds__(kThreads) void add_parts_kernel(
    const float *__restrict__ parts, const float *__restrict__ bias_parts, Groups g, uint32_t per,
    uint32_t places, int64_t weight_size, int64_t bias_size, uint32_t weight_blocks,
    uint32_t bias_blocks, T *__restrict__ v_weight, T *__restrict__ v_bias) {
  constexpr int kRun = kShare == 1 ? 4 : 1, kLanes = kThreads / kShare;
  constexpr int kElements = kLanes * kRun;
  using Run = UnalignedRun<float, kRun>;
  __shared__ float s_sum[kShare][kLanes];
  const int32_t e = static_cast<int32_t>(blockIdx.y);
  const bool is_bias = blockIdx.x >= weight_blocks;
  const int64_t size = is_bias ? bias_size : weight_size;
  uint32_t before = 0, mine = 0;
  for (int32_t e0 = 0; e0 <= e; e0 += 64) {
    const int32_t q = e0 + static_cast<int32_t>(lane_id());
    uint32_t n = 0;
    if (q <= e) {
      const int64_t rows = g.bound(q + 1) - g.bound(q);
      n = rows > 0 ? static_cast<uint32_t>((rows + per - 1) / per) : 0u;
    }
    const uint32_t end = before + wave_inclusive_scan(kept_parts(n));
    mine = readlane_u32(n, static_cast<uint32_t>(min(e - e0, 63)));
    before = readlane_u32(end, 63);
  }
  if (mine == 1) return;
  // Offsets that do not ascend could name more parts than there are places.
  const uint32_t first = min(before - mine, places);
  mine = min(mine, places - first);
  const uint32_t share = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const uint32_t block = blockIdx.x - (is_bias ? weight_blocks : 0);
  const int64_t stride = static_cast<int64_t>(is_bias ? bias_blocks : weight_blocks) * kElements;
  T *out = (is_bias ? v_bias : v_weight) + static_cast<int64_t>(e) * size;
  for (int64_t i0 = static_cast<int64_t>(block) * kElements; i0 < size; i0 += stride) {
    const int64_t i = i0 + lane * kRun;
    const float *p = (is_bias ? bias_parts : parts) + static_cast<int64_t>(first) * size + i;
    constexpr uint32_t kBatch = 8 / kRun;  // loads before their sums
    float sum[kRun] = {};
    if (i + kRun <= size) {
      for (uint32_t s = share; s < mine; s += kShare * kBatch) {
        Run v[kBatch];
#pragma unroll
        for (uint32_t q = 0; q < kBatch; ++q)
          v[q] = *reinterpret_cast<const Run *>(
              p + static_cast<int64_t>(min(s + q * kShare, mine - 1)) * size);
#pragma unroll
        for (uint32_t q = 0; q < kBatch; ++q)
#pragma unroll
          for (int r = 0; r < kRun; ++r) sum[r] += s + q * kShare < mine ? v[q].v[r] : 0.0f;
      }
    } else {
#pragma unroll
      for (int r = 0; r < kRun; ++r)
        for (uint32_t s = share; s < mine && i + r < size; s += kShare)
          sum[r] += p[static_cast<int64_t>(s) * size + r];
    }
    if constexpr (kShare > 1) {
      s_sum[share][lane] = sum[0];
      __syncthreads();
      if (share == 0) {
#pragma unroll
        for (int q = 1; q < kShare; ++q) sum[0] += s_sum[q][lane];
      }
      __syncthreads();
      if (share == 0 && i < size) out[i] = static_cast<T>(sum[0]);
    } else {
      store_run<T, kRun>(out, i, size, {f32x4{sum[0], sum[1], sum[2], sum[3]}});
    }
  }
}

// ---------------------------------------------------------------- host ---

// Bytes of the summed index per stage.  Operands read across and tiles of 128
// columns take 64: four blocks share a CU instead of two.  16k x 1024 x 1024
// bf16: input gradient 78 us with 128 bytes and 69 with 64, weights' gradient 119
// and 97; 500k x 64 x 64, where tiles have 64 columns: weights' gradient 33 and
// 37, input gradient 31 both ways.  Operands read along take 128, as runs of
// columns need (along_swizzle).
constexpr int slab_bytes(bool across, int cols) { return across && cols == 128 ? 64 : 128; }

int64_t weight_tiles(int64_t k, int64_t m) {
  return ceil_div(m, kRows) * ceil_div(std::max<int64_t>(k, 1), kRows);
}

// Rows of a part of the weights' gradient: enough parts to fill the device,
// and no more, since every part of a group past its first is a copy of the
// weight to write and add.  Blocks in all, weights' kernel and the parts' sum:
// 500k x 64 x 64 bf16 (1 tile) 39 us with 768 and 47 with 1152, 100k x 256 x 256
// (4) 54 and 66, 8000 x 512 x 512 f32 (16) 75 and 75, 28k x 256 x 1024 bf16 (16)
// 54 and 61, 16k x 1024 x 1024 (64) 120 and 110.  At least 512 rows where 16-bit products of many
// tiles take less time than that: 4000 x 1024 x 1024 bf16, forward and back,
// 73 us and 84 with 128, 28k x 256 x 1024 133 and 136; 32-bit products are slower
// and need the parts: 8000 x 512 x 512 188 us, and 208 with 512.
uint32_t rows_per_part(int64_t n, int64_t k, int64_t m, size_t element) {
  const int64_t tiles = weight_tiles(k, m);
  const int64_t even = ceil_div(n * tiles, tiles > 8 ? 1152 : 768);
  const int64_t least = tiles > 8 && element == 2 ? 512 : 128;
  return static_cast<uint32_t>(
      std::min<int64_t>(std::max<int64_t>(align_up(even, 64), least), 4096));
}

// Blocks of the weights' gradient along the rows, at most.
int64_t part_slots(int64_t n, int64_t k, int64_t m, int64_t groups, size_t element) {
  return ceil_div(n, rows_per_part(n, k, m, element)) + groups;
}

// Parts of groups that have several, at most: such a group of r rows has more
// than `per` of them, so fewer than 2 r / per parts, and fewer than r / per + 1.
int64_t part_places(int64_t n, int64_t k, int64_t m, int64_t groups, size_t element) {
  const int64_t per = rows_per_part(n, k, m, element);
  return n <= per ? 0 : std::min(2 * n / per, n / per + groups);
}

struct GradSpace {
  float *parts, *bias_parts;
};
// parts only where the weights' gradient is wanted.
GradSpace carve_grad(Carver &cv, int64_t n, int64_t k, int64_t m, int64_t groups, size_t element,
                     bool with_weight) {
  const int64_t places = part_places(n, k, m, groups, element);
  GradSpace s;
  s.parts = cv.take<float>(with_weight ? places * m * k : 0);
  s.bias_parts = cv.take<float>(std::max<int64_t>(places, 1) * m);
  return s;
}

int check_grouped(const char *what, int type, const int32_t *offsets, int64_t n, int64_t k,
                  int64_t m, int64_t groups) {
  R2S_REQUIRE(known_type(type), "%s: unknown element type %d", what, type);
  R2S_REQUIRE(n >= 0 && k >= 0 && m >= 0 && groups >= 0, "%s: negative size", what);
  R2S_REQUIRE(offsets != nullptr, "%s: null offsets", what);
  if (n > kInt32Max || k > (1 << 20) || m > (1 << 20) || groups > 65535) {
    set_error("%s: more than 2^31 - 1 rows, 2^20 columns or 65535 groups", what);
    return R2S_ERANGE;
  }
  return R2S_OK;
}

template <typename T, bool kBack, bool kVec, int kCols>
int rows_launch(const T *in, int64_t stride, const T *weight, const T *bias, Groups g,
                const int32_t *rows, int64_t k, int64_t m, T *out, hipStream_t stream) {
  const int64_t inner = kBack ? m : k, outer = kBack ? k : m;
  const int64_t col_tiles = ceil_div(outer, kCols);
  const int64_t blocks = (ceil_div(g.n, kRows) + g.count + 1) * col_tiles;
  if (blocks > kInt32Max) {
    set_error("grouped_matmul: too many tiles");
    return R2S_ERANGE;
  }
  constexpr int S = slab_bytes(kBack, kCols);
  const int stages = inner * static_cast<int64_t>(sizeof(T)) > S ? 2 : 1;
  rows_kernel<T, kBack, kVec, kCols, S>
      <<<dim3(static_cast<uint32_t>(blocks)), dim3(kThreads),
         stages * (kCols + kRows) * S, stream>>>(
          in, stride, weight, bias, g, rows, k, m, static_cast<uint32_t>(col_tiles),
          out);
  return check_launch("grouped_matmul");
}

template <typename T, bool kBack>
int rows_product(const void *in, int64_t stride, const void *weight, const void *bias, Groups g,
                 const int32_t *rows, int64_t k, int64_t m, void *out, hipStream_t stream) {
  const bool vec = address(in) % 16 == 0 && address(weight) % 16 == 0 &&
                   stride * sizeof(T) % 16 == 0 && k * sizeof(T) % 16 == 0 &&
                   (!kBack || m * sizeof(T) % 16 == 0);
  const T *ti = static_cast<const T *>(in), *tw = static_cast<const T *>(weight);
  const T *tb = static_cast<const T *>(bias);
  T *to = static_cast<T *>(out);
  // 64 columns to a tile, too, where 128 give less than one and a half blocks per
  // CU.  Forward and back: 3000 x 128 x 256 f32 49 us and 65, 4000 x 1024 x 1024
  // bf16 86 and 98; with 458 blocks (28k x 1024 x 256 bf16) 142 and 134.
  const int64_t outer = kBack ? k : m;
  const bool narrow = outer <= 64 ||
                      (ceil_div(g.n, kRows) + g.count) * ceil_div(outer, 128) <= 384;
#define R2S_ROWS(VEC, COLS) \
  return (rows_launch<T, kBack, VEC, COLS>(ti, stride, tw, tb, g, rows, k, m, to, stream))
  if (vec) {
    if (narrow) R2S_ROWS(true, 64);
    R2S_ROWS(true, 128);
  }
  if (narrow) R2S_ROWS(false, 64);
  R2S_ROWS(false, 128);
#undef R2S_ROWS
}

template <typename T, bool kVec, int kCols>
int weights_launch(const T *x, int64_t x_stride, const T *v_y, int64_t v_stride, Groups g,
                   const int32_t *rows, int64_t k, int64_t m, T *v_weight, T *v_bias,
                   const GradSpace &s, hipStream_t stream) {
  const uint32_t per = rows_per_part(g.n, k, m, sizeof(T));
  const int64_t slots = part_slots(g.n, k, m, g.count, sizeof(T));
  const uint32_t places = static_cast<uint32_t>(part_places(g.n, k, m, g.count, sizeof(T)));
  const int64_t m_tiles = ceil_div(m, kRows), k_tiles = ceil_div(std::max<int64_t>(k, 1), kCols);
  if (slots * m_tiles * k_tiles > kInt32Max) {
    set_error("grouped_matmul_bwd: too many tiles");
    return R2S_ERANGE;
  }
  if (g.n > 0) {
    constexpr int S = slab_bytes(true, kCols);
    weights_kernel<T, kVec, kCols, S>
        <<<dim3(static_cast<uint32_t>(slots * m_tiles * k_tiles)), dim3(kThreads),
           2 * (kCols + kRows) * S, stream>>>(
            x, x_stride, v_y, v_stride, g, rows, k, m, per, static_cast<uint32_t>(m_tiles),
            static_cast<uint32_t>(k_tiles), places, s.parts, s.bias_parts, v_weight, v_bias);
    R2S_RETURN_IF(check_launch("grouped_matmul_bwd weights"));
  }
  // At most 256 blocks a group: most groups of large weights have one part, and
  // their blocks only find that out.
  const bool small = m * k <= 1 << 15;
  const int64_t elements = small ? kThreads / 8 : kThreads * 4;
  const int64_t weight_blocks =
      v_weight != nullptr ? std::min<int64_t>(ceil_div(m * k, elements), 256) : 0;
  const int64_t bias_blocks = v_bias != nullptr ? ceil_div(m, elements) : 0;
  if (weight_blocks + bias_blocks == 0) return R2S_OK;
  const dim3 grid(static_cast<uint32_t>(weight_blocks + bias_blocks), g.count);
#define R2S_ADD_PARTS(SHARE)                                                                    \
  add_parts_kernel<T, SHARE><<<grid, dim3(kThreads), 0, stream>>>(                              \
      s.parts, s.bias_parts, g, per, places, m * k, m,                                          \
      static_cast<uint32_t>(weight_blocks), static_cast<uint32_t>(bias_blocks), v_weight, v_bias)
  if (small)
    R2S_ADD_PARTS(8);
  else
    R2S_ADD_PARTS(1);
#undef R2S_ADD_PARTS
  return check_launch("grouped_matmul_bwd weights");
}

template <typename T>
int weights_product(const void *x, int64_t x_stride, const void *v_y, int64_t v_stride, Groups g,
                    const int32_t *rows, int64_t k, int64_t m, void *v_weight, void *v_bias,
                    const GradSpace &s, hipStream_t stream) {
  const bool vec = k > 0 && address(x) % 16 == 0 && address(v_y) % 16 == 0 &&
                   x_stride * sizeof(T) % 16 == 0 && v_stride * sizeof(T) % 16 == 0 &&
                   k * sizeof(T) % 16 == 0 && m * sizeof(T) % 16 == 0;
  const T *tx = static_cast<const T *>(x), *tv = static_cast<const T *>(v_y);
  T *vw = static_cast<T *>(v_weight), *vb = static_cast<T *>(v_bias);
#define R2S_WEIGHTS(VEC, COLS) \
  return (weights_launch<T, VEC, COLS>(tx, x_stride, tv, v_stride, g, rows, k, m, vw, vb, s, stream))
  if (vec) {
    if (k <= 64) R2S_WEIGHTS(true, 64);
    R2S_WEIGHTS(true, 128);
  }
  if (k <= 64) R2S_WEIGHTS(false, 64);
  R2S_WEIGHTS(false, 128);
#undef R2S_WEIGHTS
}

}  // namespace
}  // namespace r2s

extern "C" {

int r2s_grouped_matmul_fwd(const void *x, int64_t x_stride, const void *weight, const void *bias,
                           const int32_t *offsets, const int32_t *rows, int64_t n, int64_t k,
                           int64_t m, int64_t groups, int32_t type, void *y, r2s_stream_t st) {
  using namespace r2s;
  clear_error();
  R2S_RETURN_IF(check_grouped("grouped_matmul_fwd", type, offsets, n, k, m, groups));
  if (n == 0 || m == 0) return R2S_OK;
  R2S_REQUIRE(x_stride >= k, "grouped_matmul_fwd: rows overlap");
  R2S_REQUIRE(y != nullptr && (k == 0 || (x != nullptr && (weight != nullptr || groups == 0))),
              "grouped_matmul_fwd: null input, weight or output");
  const Groups g{offsets, n, static_cast<int32_t>(groups)};
  R2S_BY_TYPE(type, {
    return rows_product<T, false>(x, x_stride, weight, bias, g, rows, k, m, y, as_stream(st));
  });
  return R2S_OK;
}

int64_t r2s_grouped_matmul_bwd_workspace_bytes(int64_t n, int64_t k, int64_t m, int64_t groups,
                                               int32_t type, int32_t with_weight) {
  if (n < 0 || k < 0 || m < 0 || groups < 0 || !r2s::known_type(type)) return 0;
  r2s::Carver cv(nullptr);
  r2s::carve_grad(cv, n, k, m, groups, r2s::type_size(type), with_weight != 0);
  return static_cast<int64_t>(cv.used);
}

int r2s_grouped_matmul_bwd(const void *x, int64_t x_stride, const void *weight,
                           const int32_t *offsets, const int32_t *rows, const void *v_y,
                           int64_t v_y_stride, int64_t n, int64_t k, int64_t m, int64_t groups,
                           int32_t type, void *v_x, void *v_weight, void *v_bias, void *ws,
                           size_t ws_bytes, r2s_stream_t st) {
  using namespace r2s;
  clear_error();
  R2S_RETURN_IF(check_grouped("grouped_matmul_bwd", type, offsets, n, k, m, groups));
  R2S_REQUIRE(x_stride >= k && v_y_stride >= m, "grouped_matmul_bwd: rows overlap");
  const Groups g{offsets, n, static_cast<int32_t>(groups)};
  hipStream_t stream = as_stream(st);
  if (v_x != nullptr && n > 0 && k > 0) {
    R2S_REQUIRE(m == 0 || (v_y != nullptr && (weight != nullptr || groups == 0)),
                "grouped_matmul_bwd: null gradient or weight");
    R2S_BY_TYPE(type, R2S_RETURN_IF(rows_product<T, true>(v_y, v_y_stride, weight, nullptr, g,
                                                          rows, k, m, v_x, stream)));
  }
  if ((v_weight == nullptr && v_bias == nullptr) || groups == 0 || m == 0) return R2S_OK;
  R2S_REQUIRE(n == 0 || (v_y != nullptr && (x != nullptr || k == 0)),
              "grouped_matmul_bwd: null gradient or input");
  const int64_t need =
      r2s_grouped_matmul_bwd_workspace_bytes(n, k, m, groups, type, v_weight != nullptr);
  if (ws == nullptr || static_cast<int64_t>(ws_bytes) < need) {
    set_error("grouped_matmul_bwd: workspace of %zu bytes, %lld required", ws_bytes,
              (long long)need);
    return R2S_EWORKSPACE;
  }
  Carver cv(ws);
  const GradSpace s = carve_grad(cv, n, k, m, groups, type_size(type), v_weight != nullptr);
  R2S_BY_TYPE(type, return (weights_product<T>(x, x_stride, v_y, v_y_stride, g, rows, k, m,
                                               v_weight, v_bias, s, stream)));
  return R2S_OK;
}

}  // extern "C"
