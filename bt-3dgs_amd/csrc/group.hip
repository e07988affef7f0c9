// Positions grouped by their ids: a stable radix sort of (id, position) for
// the row lookup's gradient and for the groups of a grouped product.
//
// The ids lie in [0, n_groups); any other sorts behind them.  Short lists take
// one launch (short_list_kernel), others passes of at most 9 bits (one for up to
// 511 groups, two for up to 2^18 - 1) and, after more than one, a launch for the
// offsets.  A pass cuts the list into at most kMaxTiles tiles of equal length and
// is two launches: the digit counts of every tile, then the scatter, whose blocks each add up the
// counts table themselves (at most kTableWords words, every thread a few
// dozen loads in parallel) instead of a scan between the two.  Lists this short
// are bound by launches and waits, not by bytes: 500k ids of 4096 groups,
// both passes and the offsets, take 33 us, against 51 us through the tile
// binning's sort, whose tiles, digits and lookups are made for longer lists.
#include <algorithm>

#include "r2s_latent.h"
#include "r2s_scan.h"

namespace r2s {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kRounds = 4;                    // items per thread and subtile
constexpr int kSubtile = kThreads * kRounds;
constexpr uint32_t kMaxBits = 9;
constexpr int kMaxDigits = 1 << kMaxBits;
constexpr int64_t kMaxTiles = 256, kTableWords = 32768;
static_assert(kMaxDigits <= kThreads, "one digit per thread in the scans");

// An input id as a sort key: itself, or n_groups where it names no group.
template <typename I>
__device__ __forceinline__ uint32_t sort_key(I id, uint32_t n_groups) {
  if constexpr (std::is_same<I, uint32_t>::value)
    return id;  // a key of an earlier pass
  else
    return id >= 0 && static_cast<uint64_t>(id) < n_groups ? static_cast<uint32_t>(id) : n_groups;
}

// table [tiles][digits]: each tile's count of each digit.
template <typename I>
__global__ __launch_bounds__(kThreads) void digit_count_kernel(const I *__restrict__ ids,
                                                               int64_t n, int64_t tile_items,
                                                               uint32_t n_groups, uint32_t shift,
                                                               uint32_t bits,
                                                               uint32_t *__restrict__ table) {
  __shared__ uint32_t count[kMaxDigits];
  const uint32_t digits = 1u << bits, mask = digits - 1u;
  if (threadIdx.x < digits) count[threadIdx.x] = 0;
  __syncthreads();
  const int64_t begin = blockIdx.x * tile_items, end = min(begin + tile_items, n);
  for (int64_t i0 = begin; i0 < end; i0 += kSubtile) {
    uint32_t key[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
      key[r] = sort_key(ids[min(i0 + r * kThreads + threadIdx.x, end - 1)], n_groups);
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
      if (i0 + r * kThreads + threadIdx.x < end) atomicAdd(&count[(key[r] >> shift) & mask], 1u);
  }
  __syncthreads();
  if (threadIdx.x < digits) table[blockIdx.x * digits + threadIdx.x] = count[threadIdx.x];
}

// Moves each item to its place of the pass.  order_in null: the first pass,
// whose positions are the indices.  keys_out may be null (the last pass);
// offsets (null unless this is the only pass) receives the digits' starts.
template <typename I>
__global__ __launch_bounds__(kThreads) void digit_scatter_kernel(
    const I *__restrict__ ids, const uint32_t *__restrict__ order_in, int64_t n,
    int64_t tile_items, uint32_t n_groups, uint32_t shift, uint32_t bits, uint32_t tiles,
    const uint32_t *__restrict__ table, uint32_t *__restrict__ keys_out,
    uint32_t *__restrict__ order_out, int32_t *__restrict__ offsets) {
  __shared__ uint32_t s_all[kThreads], s_before[kThreads];
  __shared__ uint32_t base[kMaxDigits];          // the next free place of each digit
  __shared__ uint32_t count[kWaves][kMaxDigits];  // per wave, then each wave's first place
  __shared__ uint32_t s_scan[kWaves];
  const uint32_t digits = 1u << bits, mask = digits - 1u;
  const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  {
    // Digit d's first place for this tile: the items of smaller digits, and
    // those of digit d in the tiles before.  kThreads / digits threads per digit
    // share the tiles.
    const uint32_t d = threadIdx.x & mask, part = threadIdx.x >> bits, parts = kThreads >> bits;
    uint32_t all = 0, before = 0;
    for (uint32_t t0 = part; t0 < tiles; t0 += parts * 16) {
      uint32_t v[16];
#pragma unroll
      for (uint32_t k = 0; k < 16; ++k)
        v[k] = table[min(t0 + k * parts, tiles - 1) * digits + d];
#pragma unroll
      for (uint32_t k = 0; k < 16; ++k) {
        const uint32_t t = t0 + k * parts, x = t < tiles ? v[k] : 0u;
        all += x;
        before += t < blockIdx.x ? x : 0u;
      }
    }
    s_all[threadIdx.x] = all;
    s_before[threadIdx.x] = before;
    __syncthreads();
    all = before = 0;
    if (threadIdx.x < digits) {
      for (uint32_t p = 0; p < parts; ++p) {
        all += s_all[(p << bits) + threadIdx.x];
        before += s_before[(p << bits) + threadIdx.x];
      }
    }
    uint32_t total;
    const uint32_t start = block_exclusive_scan(all, s_scan, total);
    if (threadIdx.x < digits) base[threadIdx.x] = start + before;
    if (offsets != nullptr && blockIdx.x == 0 && threadIdx.x <= n_groups &&
        threadIdx.x < digits)
      offsets[threadIdx.x] = static_cast<int32_t>(start);
  }
  const uint64_t lower = lanemask_lt();
  const int64_t begin = blockIdx.x * tile_items, end = min(begin + tile_items, n);
  for (int64_t i0 = begin; i0 < end; i0 += kSubtile) {
    // Wave w has the w-th run of the subtile, so (wave, round, lane) is the
    // order of the items.
    const int64_t first = i0 + wave * (64 * kRounds) + lane;
    uint32_t key[kRounds], pos[kRounds], rank[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const int64_t i = min(first + r * 64, end - 1);
      key[r] = sort_key(ids[i], n_groups);
      pos[r] = order_in != nullptr ? order_in[i] : static_cast<uint32_t>(i);
    }
    for (uint32_t k = lane; k < digits; k += 64) count[wave][k] = 0;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const bool valid = first + r * 64 < end;
      const uint32_t d = (key[r] >> shift) & mask;
      uint64_t peers = ballot(valid);
      // Lanes whose digit differs in some bit; bits at or above `bits` are zero
      // in every digit, so they mark none.
      uint64_t differ = 0;
#pragma unroll
      for (uint32_t b = 0; b < kMaxBits; ++b) {
        const uint32_t x =
            static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int32_t>(d), b, 1));
        differ |= ballot(x != 0u) ^ ((static_cast<uint64_t>(x) << 32) | x);
      }
      peers &= ~differ;
      const uint32_t c = count[wave][d];
      rank[r] = c + static_cast<uint32_t>(__popcll(peers & lower));
      // The highest lane of each digit moves the digit's counter on.
      if (valid && lane == 63u - static_cast<uint32_t>(__clzll(peers)))
        count[wave][d] = c + static_cast<uint32_t>(__popcll(peers));
    }
    __syncthreads();
    if (threadIdx.x < digits) {
      uint32_t run = base[threadIdx.x];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const uint32_t c = count[w][threadIdx.x];
        count[w][threadIdx.x] = run;
        run += c;
      }
      base[threadIdx.x] = run;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      if (first + r * 64 < end) {
        const uint32_t at = count[wave][(key[r] >> shift) & mask] + rank[r];
        if (keys_out != nullptr) keys_out[at] = key[r];
        order_out[at] = pos[r];
      }
    }
  }
}

// offsets[v] = the first sorted key that is at least v, for v <= n_groups: the
// thread of entry i writes it for the ids after the entry before, up to its own
// (the thread past the end: up to n_groups).  A wave fills long gaps together,
// so that a few ids far apart cost no thread a walk over all of them.
__global__ __launch_bounds__(256) void group_offsets_kernel(const uint32_t *__restrict__ keys,
                                                            uint32_t n, uint32_t n_groups,
                                                            int32_t *__restrict__ offsets) {
  const uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
  // [from, to): the ids whose first entry is i.
  uint32_t from = 0, to = 0;
  if (i <= n) {
    if (i > 0) from = keys[i - 1] + 1;
    to = i < n ? keys[i] + 1 : n_groups + 1;
  }
  constexpr uint32_t kShort = 16;
  uint64_t wide = ballot(to > from && to - from > kShort);
  if (to > from && to - from <= kShort)
    for (uint32_t v = from; v < to; ++v) offsets[v] = static_cast<int32_t>(i);
  while (wide != 0) {
    const uint32_t src =
        static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(wide))) - 1u;
    wide &= wide - 1;
    const uint32_t a = readlane_u32(from, src), b = readlane_u32(to, src);
    const int32_t at = static_cast<int32_t>(readlane_u32(static_cast<uint32_t>(i), src));
    for (uint32_t v = a + lane_id(); v < b; v += 64) offsets[v] = at;
  }
}

// A short list in one launch: every item counts the items that go before it, and
// every group those of the groups before it, over the keys in LDS.  kShare lanes
// take a part of the keys each: with one, 2000 items took 43 us.
constexpr int kShortThreads = 256, kShortList = 4096, kShare = 8;
constexpr int kShortItems = kShortThreads / kShare;  // of a block
template <typename I>
__global__ __launch_bounds__(kShortThreads) void short_list_kernel(
    const I *__restrict__ ids, int32_t n, uint32_t n_groups, uint32_t item_blocks,
    uint32_t *__restrict__ keys_out, int32_t *__restrict__ order, int32_t *__restrict__ offsets) {
  __shared__ __attribute__((aligned(16))) uint32_t s_key[kShortList];
  constexpr int kStep = 4 * kShare;  // keys of a turn
  const int32_t padded = (n + kStep - 1) / kStep * kStep;
  for (int32_t j = static_cast<int32_t>(threadIdx.x); j < padded; j += kShortThreads)
    s_key[j] = j < n ? sort_key(ids[j], n_groups) : ~0u;
  __syncthreads();
  const bool group = blockIdx.x >= item_blocks;
  const uint32_t i = (blockIdx.x - (group ? item_blocks : 0u)) * kShortItems + threadIdx.x / kShare;
  const bool some = i < (group ? n_groups + 1u : static_cast<uint32_t>(n));
  const uint32_t mine = group ? i : s_key[some ? i : 0u];
  const int32_t at = group ? 0 : static_cast<int32_t>(i);  // equal keys before it count
  int32_t before = 0;
#pragma unroll 4
  for (int32_t j = static_cast<int32_t>(threadIdx.x % kShare) * 4; j < padded; j += kStep) {
    const uint4 k = *reinterpret_cast<const uint4 *>(s_key + j);
    before += (k.x < mine + (j < at)) + (k.y < mine + (j + 1 < at)) +
              (k.z < mine + (j + 2 < at)) + (k.w < mine + (j + 3 < at));
  }
#pragma unroll
  for (int off = 1; off < kShare; off *= 2) before += __shfl_xor(before, off, 64);
  if (!some || threadIdx.x % kShare != 0) return;
  if (group) {
    offsets[i] = before;
  } else {
    order[before] = static_cast<int32_t>(i);
    if (keys_out != nullptr) keys_out[before] = mine;
  }
}

// ---------------------------------------------------------------- host ---

// Whether a list goes through short_list_kernel, whose work is n (n + groups).
// A lookup and its gradient, 64 columns: 4000 ids of 4096 rows 28 us and 36 in
// passes, of 500 rows (one pass) 28 and 29, 264 ids of 108k rows 28 and 56; 8000
// ids of 100 rows 38 and 29, and with four times the work of this limit, 2000 ids
// of 120k rows, 53 and 41.
bool is_short(int64_t n, int64_t n_groups) {
  return n <= kShortList && n * (n + n_groups) <= (1 << 26);
}

struct Sizes {
  uint32_t passes, bits;  // bits of every pass but the last, which has the rest
  uint32_t key_bits;
  int64_t tile_items, tiles;
};

Sizes sizes_of(int64_t n, int64_t n_groups) {
  Sizes s{};
  s.key_bits = 1;
  while (s.key_bits < 32 && (int64_t{1} << s.key_bits) < n_groups + 1) ++s.key_bits;
  s.passes = (s.key_bits + kMaxBits - 1) / kMaxBits;
  s.bits = (s.key_bits + s.passes - 1) / s.passes;
  const int64_t most = std::min(kMaxTiles, kTableWords >> s.bits);
  s.tile_items = std::max<int64_t>(ceil_div(n, most), kThreads);
  s.tiles = ceil_div(n, s.tile_items);
  return s;
}

struct GroupSpace {
  uint32_t *table, *keys[2], *order[2];
};

GroupSpace carve_group(Carver &cv, int64_t n, const Sizes &z, bool own_keys) {
  GroupSpace s{};
  s.table = cv.take<uint32_t>(z.tiles << z.bits);
  for (int i = 0; i < 2; ++i) {
    // The passes before the last write to one pair, then the other.
    const bool used = static_cast<uint32_t>(i) + 1 < z.passes;
    s.keys[i] = cv.take<uint32_t>(used ? n : 0);
    s.order[i] = cv.take<uint32_t>(used ? n : 0);
  }
  if (own_keys && z.passes > 1) s.keys[(z.passes - 1) % 2] = cv.take<uint32_t>(n);
  return s;
}

template <typename I>
int pass(const I *ids, const uint32_t *order_in, int64_t n, uint32_t n_groups, const Sizes &z,
         uint32_t p, uint32_t *table, uint32_t *keys_out, uint32_t *order_out, int32_t *offsets,
         hipStream_t stream) {
  const uint32_t shift = p * z.bits, bits = std::min(z.bits, z.key_bits - shift);
  const dim3 grid(static_cast<uint32_t>(z.tiles)), block(kThreads);
  digit_count_kernel<I><<<grid, block, 0, stream>>>(ids, n, z.tile_items, n_groups, shift, bits,
                                                    table);
  R2S_RETURN_IF(check_launch("group_rows count"));
  digit_scatter_kernel<I><<<grid, block, 0, stream>>>(
      ids, order_in, n, z.tile_items, n_groups, shift, bits, static_cast<uint32_t>(z.tiles),
      table, keys_out, order_out, offsets);
  return check_launch("group_rows scatter");
}

}  // namespace

int64_t sort_ids_bytes(int64_t n, int64_t n_groups) {
  if (n <= 0) return 0;
  Carver cv(nullptr);
  carve_group(cv, n, sizes_of(n, n_groups), true);
  return static_cast<int64_t>(cv.used);
}

int sort_ids(const void *ids, bool wide, int64_t n, int64_t n_groups, int32_t *order,
             int32_t *offsets, uint32_t *keys, void *workspace, hipStream_t stream) {
  if (n == 0)
    return offsets == nullptr
               ? R2S_OK
               : device_fill<int32_t>(offsets, n_groups + 1, 0, stream, "group_rows");
  if (is_short(n, n_groups)) {
    const uint32_t items = static_cast<uint32_t>(ceil_div(n, kShortItems));
    const dim3 grid(items + (offsets != nullptr ? static_cast<uint32_t>(
                                                      ceil_div(n_groups + 1, kShortItems))
                                                : 0u));
    const int32_t count = static_cast<int32_t>(n);
    const uint32_t groups = static_cast<uint32_t>(n_groups);
    if (wide)
      short_list_kernel<<<grid, dim3(kShortThreads), 0, stream>>>(
          static_cast<const int64_t *>(ids), count, groups, items, keys, order, offsets);
    else
      short_list_kernel<<<grid, dim3(kShortThreads), 0, stream>>>(
          static_cast<const int32_t *>(ids), count, groups, items, keys, order, offsets);
    return check_launch("group_rows short list");
  }
  const Sizes z = sizes_of(n, n_groups);
  Carver cv(workspace);
  GroupSpace s = carve_group(cv, n, z, keys == nullptr);
  const uint32_t g = static_cast<uint32_t>(n_groups);
  const uint32_t *kin = nullptr, *oin = nullptr;
  for (uint32_t p = 0; p < z.passes; ++p) {
    const bool last = p + 1 == z.passes;
    // A caller's keys, or the workspace's where the offsets are searched in them.
    uint32_t *kout = !last ? s.keys[p % 2] : keys != nullptr ? keys : z.passes > 1 ? s.keys[p % 2]
                                                                                   : nullptr;
    uint32_t *oout = last ? reinterpret_cast<uint32_t *>(order) : s.order[p % 2];
    int32_t *starts = z.passes == 1 ? offsets : nullptr;
    if (p > 0)
      R2S_RETURN_IF(pass(kin, oin, n, g, z, p, s.table, kout, oout, starts, stream));
    else if (wide)
      R2S_RETURN_IF(pass(static_cast<const int64_t *>(ids), oin, n, g, z, p, s.table, kout, oout,
                         starts, stream));
    else
      R2S_RETURN_IF(pass(static_cast<const int32_t *>(ids), oin, n, g, z, p, s.table, kout, oout,
                         starts, stream));
    kin = kout;
    oin = oout;
  }
  if (offsets == nullptr || z.passes == 1) return R2S_OK;
  group_offsets_kernel<<<dim3(static_cast<uint32_t>(ceil_div(n + 1, 256))), dim3(256), 0,
                         stream>>>(kin, static_cast<uint32_t>(n), g, offsets);
  return check_launch("group_rows offsets");
}

}  // namespace r2s

extern "C" {

int64_t r2s_group_rows_workspace_bytes(int64_t n, int64_t n_groups) {
  return n > 0 && n_groups >= 0 ? r2s::sort_ids_bytes(n, n_groups) : 0;
}

int r2s_group_rows(const void *ids, int32_t ids_are_64, int64_t n, int64_t n_groups,
                   int32_t *rows, int32_t *offsets, void *ws, size_t ws_bytes, r2s_stream_t st) {
  using namespace r2s;
  clear_error();
  R2S_REQUIRE(n >= 0 && n_groups >= 0, "group_rows: negative size");
  if (n > kInt32Max || n_groups >= kInt32Max) {
    set_error("group_rows: more than 2^31 - 1 rows or groups");
    return R2S_ERANGE;
  }
  R2S_REQUIRE(offsets != nullptr && (n == 0 || (ids != nullptr && rows != nullptr)),
              "group_rows: null ids, rows or offsets");
  const int64_t need = r2s_group_rows_workspace_bytes(n, n_groups);
  if (need > 0 && (ws == nullptr || static_cast<int64_t>(ws_bytes) < need)) {
    set_error("group_rows: workspace of %zu bytes, %lld required", ws_bytes, (long long)need);
    return R2S_EWORKSPACE;
  }
  return sort_ids(ids, ids_are_64 != 0, n, n_groups, rows, offsets, nullptr, ws, as_stream(st));
}

}  // extern "C"
