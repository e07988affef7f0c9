// Rows of a table by id, scaled, and the table's gradient.
//
//   forward   out_i = s T[id_i]: each thread moves vectors of 16 bytes, at any
//             element.  Ids outside the table give zero
//             rows, so no id reads out of range.
//   backward  dT_v = s sum_{id_i = v} dy_i, without atomics: the positions are
//             sorted by id (stable, group.hip), the sorted list is cut into
//             chunks of equal length whatever the ids are, and each chunk sums
//             its runs of equal ids in float32.  A run inside one chunk is a
//             finished row; a run that crosses chunk ends leaves one partial
//             row per chunk, and a second kernel adds those in chunk order and
//             writes the rows that no id names as zeros.  Chunks keep the work
//             even when a few ids own almost every position, and fix the order
//             of the sums.
#include <algorithm>

#include "r2s_latent.h"

namespace r2s {
namespace {

constexpr int kThreads = 256;

// V consecutive elements at any element, as one load or store.  Rows are taken
// in vectors of at most 16 bytes, the last of which ends with the row and may
// overlap the one before: both then hold and write the same values.  300k x 45
// f32, forward and back: 54 us, and 64 us with the vectors that divide a row;
// 200k x 99 bf16 53 and 68.
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Run {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Run<T, V> load_run(const T *p) {
  return *reinterpret_cast<const Run<T, V> *>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store_run(T *p, const Run<T, V> &x) {
  *reinterpret_cast<Run<T, V> *>(p) = x;
}

// ------------------------------------------------------------- forward ---

// Vectors per thread: as many bytes of the narrow ones.
constexpr int fwd_vectors(int bytes) { return bytes <= 4 ? 8 : 4; }

// A block takes `rows` whole rows (of at most kThreads fwd_vectors vectors
// together), or in a longer row one run of that many.  vpr: vectors per row;
// magic: 2^32 / vpr rounded up, the quotient of every vector number of a block
// (below 2^13, so exact) by one multiplication; a row of one vector, whose magic
// would be 2^32, needs none.  Bound by the writes: 64 MB of 500k x 64 bf16 rows
// in 16 us, 3.9 TB/s.
template <typename T, int V, typename I>
__global__ __launch_bounds__(kThreads) void lookup_fwd_kernel(
    const T *__restrict__ table, int64_t stride, const I *__restrict__ ids, float scale,
    int64_t n, int64_t n_rows, uint32_t width, uint32_t vpr, uint32_t rows, uint32_t magic,
    T *__restrict__ out) {
  constexpr int kVectors = fwd_vectors(V * sizeof(T));
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows;
  const uint32_t vec0 = blockIdx.y * (kThreads * kVectors);
  const uint32_t count = static_cast<uint32_t>(min(static_cast<int64_t>(rows), n - row0));
  int64_t id[kVectors], at[kVectors];
  uint32_t col[kVectors];
#pragma unroll
  for (int k = 0; k < kVectors; ++k) {
    const uint32_t q = k * kThreads + threadIdx.x;
    const uint32_t r = vpr == 1 ? q : rows > 1 ? __umulhi(q, magic) : 0u;
    const uint32_t vec = vec0 + q - r * vpr;
    const bool inside = r < count && vec < vpr;
    col[k] = min(vec * V, width - V);
    at[k] = inside ? (row0 + r) * width + col[k] : -1;
    id[k] = inside ? static_cast<int64_t>(ids[row0 + r]) : -1;
  }
  Run<T, V> x[kVectors];
#pragma unroll
  for (int k = 0; k < kVectors; ++k) {
    if (id[k] >= 0 && id[k] < n_rows) {
      x[k] = load_run<T, V>(table + id[k] * stride + col[k]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) x[k].v[j] = static_cast<T>(0.0f);
    }
  }
#pragma unroll
  for (int k = 0; k < kVectors; ++k) {
    if (at[k] >= 0) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        x[k].v[j] = static_cast<T>(static_cast<float>(x[k].v[j]) * scale);
      store_run<T, V>(out + at[k], x[k]);
    }
  }
}

// ------------------------------------------------------------ backward ---

// Threads of the second kernel's blocks: a long row of narrow vectors needs the
// more lane groups (300k ids of 18 rows of 45 f32, forward and back: 59 us with
// 1024 threads, 67 with 512), wide vectors the less LDS (64 bf16 columns: 7 us
// with 512, 14 with 1024).
constexpr int row_threads(int V) { return V <= 4 ? 1024 : 512; }
constexpr int kLongRow = 32;       // chunks: longer rows are added by a whole block
// Lanes that the chunks are spread over: the same call 54 us, and 59 with twice
// as many, whose parts are twice as many too; 50k x 297 f32 73 and 70.
constexpr int64_t kSpread = 1 << 17;

// The sorted ids (n_rows for those outside the table), their positions and each
// row's first entry.
struct Sorted {
  const uint32_t *keys;
  const int32_t *order, *offsets;
  uint32_t n;
  uint32_t chunk;  // entries per chunk
};

// 2^lane_bits lanes hold one row's columns [c0, c0 + lanes V) and walk one
// chunk; partial [chunks][2][width]: slot 0 the chunk's part of a run that began
// in an earlier chunk, slot 1 its part of one that goes on into the next (a run
// that does both is in slot 0).  500k x 64 bf16: 20 us, 64 MB of gathered rows at
// 3.2 TB/s, bound by the chain of a chunk: its ids, its positions, its rows.
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void lookup_bwd_chunks_kernel(
    const T *__restrict__ v_out, int64_t stride, Sorted list, float scale, uint32_t n_rows,
    uint32_t width, uint32_t lane_bits, T *__restrict__ v_table, float *__restrict__ partial) {
  const uint32_t vec = (blockIdx.y << lane_bits) + (threadIdx.x & ((1u << lane_bits) - 1u));
  const uint32_t col = min(vec * V, width - V);
  const uint64_t chunk = (static_cast<uint64_t>(blockIdx.x) << (8 - lane_bits)) +
                         (threadIdx.x >> lane_bits);
  const uint64_t begin = chunk * list.chunk;
  if (begin >= list.n || vec * V >= width) return;
  const uint32_t j0 = static_cast<uint32_t>(begin);
  const uint32_t j1 = static_cast<uint32_t>(min(begin + list.chunk, uint64_t{list.n}));
  // No id is n_rows + 1: nothing runs past the list's ends.
  const uint32_t before = j0 > 0 ? list.keys[j0 - 1] : n_rows + 1;
  const uint32_t after = j1 < list.n ? list.keys[j1] : n_rows + 1;
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.0f;
  uint32_t run = list.keys[j0];
  bool first = true;  // the run that began at j0
  auto flush = [&](bool last) {
    if (run == n_rows) return;
    if ((first && run == before) || (last && run == after)) {
      const int slot = first && run == before ? 0 : 1;
      float *p = partial + (chunk * 2 + slot) * width + col;
#pragma unroll
      for (int v = 0; v < V; ++v) p[v] = acc[v];
    } else {
      Run<T, V> r;
#pragma unroll
      for (int v = 0; v < V; ++v) r.v[v] = static_cast<T>(acc[v] * scale);
      store_run<T, V>(v_table + static_cast<int64_t>(run) * width + col, r);
    }
  };
  // Rows loaded before their first use: as many bytes of the narrow vectors.
  constexpr int kInFlight = sizeof(T) * V <= 4 ? 16 : 8;
  for (uint32_t j = j0; j < j1; j += kInFlight) {
    uint32_t id[kInFlight];
    Run<T, V> x[kInFlight];
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      const uint32_t i = min(j + k, j1 - 1);
      id[k] = list.keys[i];
      x[k] = load_run<T, V>(v_out + static_cast<int64_t>(list.order[i]) * stride + col);
    }
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      if (j + k < j1) {
        if (id[k] != run) {
          flush(false);
          run = id[k];
          first = false;
#pragma unroll
          for (int v = 0; v < V; ++v) acc[v] = 0.0f;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] += static_cast<float>(x[k].v[v]);
      }
    }
  }
  flush(true);
}

// acc += the parts of chunks c, c + step, ... up to `last` of a row whose first
// chunk is `first`.
template <int V>
__device__ __forceinline__ void add_parts(const float *__restrict__ partial, uint32_t width,
                                          uint32_t col, uint32_t first, uint32_t c, uint32_t last,
                                          uint32_t step, float (&acc)[V]) {
  constexpr int kParts = V <= 2 ? 16 : 8;  // loaded before their first use
  for (; c <= last; c += step * kParts) {
    float p[kParts][V];
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
      const uint32_t i = min(c + k * step, last);
      const float *q = partial + (uint64_t{i} * 2 + (i == first ? 1 : 0)) * width + col;
#pragma unroll
      for (int v = 0; v < V; ++v) p[k][v] = q[v];
    }
#pragma unroll
    for (int k = 0; k < kParts; ++k)
      if (c + k * step <= last) {
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] += p[k][v];
      }
  }
}

// Blocks from n_long on: one row per lane group -- zeros without an entry,
// the sum of its parts if it crosses a chunk end, nothing to do otherwise.
// Blocks before: block b looks at the row that holds the first entry of chunk
// (b + 1) kLongRow and adds its parts if it spans more than kLongRow chunks
// and no smaller b sees it.  200k x 256 bf16 rows, most of them zeros: 29 us, 100
// MB written at 3.6 TB/s; 18 x 45 f32 rows of 300k entries: 15 us, bound by the
// parts of the longest row.
template <typename T, int V>
__global__ __launch_bounds__(row_threads(V)) void lookup_bwd_rows_kernel(
    Sorted list, float scale, uint32_t n_rows, uint32_t width, uint32_t lane_bits,
    uint32_t n_long, const float *__restrict__ partial, T *__restrict__ v_table) {
  const uint32_t lane = threadIdx.x & ((1u << lane_bits) - 1u), group = threadIdx.x >> lane_bits;
  constexpr int kRowThreads = row_threads(V);
  const uint32_t groups = kRowThreads >> lane_bits;
  const uint32_t vec = (blockIdx.y << lane_bits) + lane;
  const uint32_t col = min(vec * V, width - V);
  const bool inside = vec * V < width;
  __shared__ float sums[kRowThreads * V];
  const bool whole = blockIdx.x < n_long;
  uint32_t row;
  if (whole) {
    const uint64_t j = (uint64_t{blockIdx.x} + 1) * kLongRow * list.chunk;
    row = list.keys[j];  // j < n: see n_long
    if (row == n_rows) return;
  } else {
    row = (blockIdx.x - n_long) * groups + group;
    if (row >= n_rows) return;
  }
  const uint32_t o0 = static_cast<uint32_t>(list.offsets[row]);
  const uint32_t o1 = static_cast<uint32_t>(list.offsets[row + 1]);
  const uint32_t c0 = o0 / list.chunk, c1 = o1 > o0 ? (o1 - 1) / list.chunk : c0;
  const bool is_long = c1 - c0 > kLongRow;
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.0f;
  if (whole) {
    // Uniform over the block: every thread of a block has the same row.
    const uint64_t smaller = uint64_t{blockIdx.x} * kLongRow * list.chunk;
    if (!is_long || (blockIdx.x > 0 && o0 <= smaller)) return;
    if (inside) add_parts<V>(partial, width, col, c0, c0 + group, c1, groups, acc);
#pragma unroll
    for (int v = 0; v < V; ++v) sums[threadIdx.x * V + v] = acc[v];
    __syncthreads();
    if (group != 0) return;
    for (uint32_t g = 1; g < groups; ++g) {
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += sums[((g << lane_bits) + lane) * V + v];
    }
  } else {
    if (o1 > o0 && (c0 == c1 || is_long)) return;
    if (inside && o1 > o0) add_parts<V>(partial, width, col, c0, c0, c1, 1, acc);
  }
  if (!inside) return;
  Run<T, V> r;
#pragma unroll
  for (int v = 0; v < V; ++v) r.v[v] = static_cast<T>(acc[v] * scale);
  store_run<T, V>(v_table + static_cast<int64_t>(row) * width + col, r);
}

// ---------------------------------------------------------------- host ---

// Entries per chunk, for rows of `lanes` lanes: as many chunks as keep the
// device busy and no more, since a row of many entries has a part per chunk to
// add afterwards.  With the fewest lanes that a width can have (16-byte
// vectors), the most chunks, which the workspace has to hold.
uint32_t chunk_entries(int64_t n, int64_t lanes) {
  const int64_t even = ceil_div(n * lanes, kSpread);
  return static_cast<uint32_t>(std::min<int64_t>(std::max<int64_t>(align_up(even, 8), 16), 1024));
}
int64_t most_chunks(int64_t n, int64_t width) {
  return ceil_div(n, chunk_entries(n, std::max<int64_t>(width / 8, 1)));
}

struct BwdSpace {
  int32_t *order, *offsets;
  uint32_t *keys;
  float *partial;
  char *sort;
};

BwdSpace carve_bwd(Carver &cv, int64_t n, int64_t n_rows, int64_t width) {
  BwdSpace s;
  s.order = cv.take<int32_t>(n);
  s.offsets = cv.take<int32_t>(n_rows + 1);
  s.keys = cv.take<uint32_t>(n);
  s.partial = cv.take<float>(most_chunks(n, width) * 2 * width);
  s.sort = cv.take<char>(sort_ids_bytes(n, n_rows));
  return s;
}

int check_lookup(const char *what, int64_t n, int64_t n_rows, int64_t width, int64_t stride,
                 int type, const void *ids) {
  R2S_REQUIRE(known_type(type), "%s: unknown element type %d", what, type);
  R2S_REQUIRE(n >= 0 && n_rows >= 0 && width >= 0, "%s: negative size", what);
  R2S_REQUIRE(stride >= width, "%s: a row stride of %lld for rows of %lld", what,
              (long long)stride, (long long)width);
  R2S_REQUIRE(n == 0 || ids != nullptr, "%s: null ids", what);
  if (n > kInt32Max || n_rows >= kInt32Max || width > (1 << 24)) {
    set_error("%s: more than 2^31 - 1 ids or rows, or rows of more than 2^24", what);
    return R2S_ERANGE;
  }
  return R2S_OK;
}

template <typename T, int V, typename I>
int lookup_fwd(const void *table, int64_t stride, const void *ids, float scale, int64_t n,
               int64_t n_rows, int64_t width, void *out, hipStream_t stream) {
  constexpr int64_t per_block = kThreads * fwd_vectors(V * static_cast<int>(sizeof(T)));
  static_assert(per_block <= 4096, "vector numbers of a block below 2^13");
  const int64_t vpr = ceil_div(width, V);
  const int64_t rows = std::max<int64_t>(per_block / vpr, 1), slices = ceil_div(vpr, per_block);
  if (ceil_div(n, rows) > kInt32Max || slices > 65535) {
    set_error("embedding_fwd: output too large");
    return R2S_ERANGE;
  }
  const uint32_t magic =
      rows > 1 && vpr > 1 ? static_cast<uint32_t>(((uint64_t{1} << 32) + vpr - 1) / vpr) : 0u;
  lookup_fwd_kernel<T, V, I>
      <<<dim3(static_cast<uint32_t>(ceil_div(n, rows)), static_cast<uint32_t>(slices)),
         dim3(kThreads), 0, stream>>>(static_cast<const T *>(table), stride,
                                      static_cast<const I *>(ids), scale, n, n_rows,
                                      static_cast<uint32_t>(width), static_cast<uint32_t>(vpr),
                                      static_cast<uint32_t>(rows), magic, static_cast<T *>(out));
  return check_launch("embedding_fwd");
}

template <typename T, int V>
int lookup_bwd(const void *v_out, int64_t stride, float scale, int64_t n, int64_t n_rows,
               int64_t width_, void *v_table_, const BwdSpace &s, hipStream_t stream) {
  T *v_table = static_cast<T *>(v_table_);
  const uint32_t width = static_cast<uint32_t>(width_), vpr = (width + V - 1) / V;
  uint32_t bits = 0;
  while (bits < 6 && (1u << bits) < vpr) ++bits;
  const uint32_t slices = static_cast<uint32_t>(ceil_div(vpr, 1 << bits));
  const Sorted list{s.keys, s.order, s.offsets, static_cast<uint32_t>(n),
                    chunk_entries(n, int64_t{slices} << bits)};
  const int64_t chunks = ceil_div(n, list.chunk);
  if (n > 0) {
    lookup_bwd_chunks_kernel<T, V>
        <<<dim3(static_cast<uint32_t>(ceil_div(chunks, kThreads >> bits)), slices),
           dim3(kThreads), 0, stream>>>(static_cast<const T *>(v_out), stride, list, scale,
                                        static_cast<uint32_t>(n_rows), width, bits, v_table,
                                        s.partial);
    R2S_RETURN_IF(check_launch("embedding_bwd"));
  }
  // Block b < n_long reads entry (b + 1) kLongRow chunk, the first of a chunk
  // that there is.
  const int64_t n_long = chunks > 0 ? (chunks - 1) / kLongRow : 0;
  lookup_bwd_rows_kernel<T, V>
      <<<dim3(static_cast<uint32_t>(n_long + ceil_div(n_rows, row_threads(V) >> bits)),
              slices),
         dim3(row_threads(V)), 0, stream>>>(list, scale, static_cast<uint32_t>(n_rows), width, bits,
                                         static_cast<uint32_t>(n_long), s.partial, v_table);
  return check_launch("embedding_bwd rows");
}

// Bytes of the vectors of a row: 16, or the power of two that a shorter row has.
int run_bytes(int64_t width, int size) {
  int bytes = 16;
  while (bytes > width * size) bytes /= 2;
  return bytes;
}

// `call` with V bound to the elements of a vector of `bytes` bytes.
#define R2S_BY_VECTOR(T, bytes, ...)                        \
  do {                                                      \
    if ((bytes) == 16) {                                    \
      constexpr int V = 16 / static_cast<int>(sizeof(T));   \
      __VA_ARGS__;                                          \
    } else if ((bytes) == 8) {                              \
      constexpr int V = 8 / static_cast<int>(sizeof(T));    \
      __VA_ARGS__;                                          \
    } else if ((bytes) == 4 || sizeof(T) == 4) {            \
      constexpr int V = 4 / static_cast<int>(sizeof(T));    \
      __VA_ARGS__;                                          \
    } else {                                                \
      constexpr int V = 1;                                  \
      __VA_ARGS__;                                          \
    }                                                       \
  } while (0)

}  // namespace
}  // namespace r2s

extern "C" {

int r2s_embedding_fwd(const void *table, int64_t table_stride, const void *ids,
                      int32_t ids_are_64, float scale, int32_t type, int64_t n, int64_t n_rows,
                      int64_t width, void *out, r2s_stream_t st) {
  using namespace r2s;
  clear_error();
  R2S_RETURN_IF(check_lookup("embedding_fwd", n, n_rows, width, table_stride, type, ids));
  if (n == 0 || width == 0) return R2S_OK;
  R2S_REQUIRE((table != nullptr || n_rows == 0) && out != nullptr,
              "embedding_fwd: null table or output");
  const int bytes = run_bytes(width, type_size(type));
  hipStream_t stream = as_stream(st);
  R2S_BY_TYPE(type, R2S_BY_VECTOR(T, bytes, {
    return ids_are_64 ? (lookup_fwd<T, V, int64_t>(table, table_stride, ids, scale, n, n_rows,
                                                   width, out, stream))
                      : (lookup_fwd<T, V, int32_t>(table, table_stride, ids, scale, n, n_rows,
                                                   width, out, stream));
  }));
  return R2S_OK;
}

int64_t r2s_embedding_bwd_workspace_bytes(int64_t n, int64_t n_rows, int64_t width) {
  if (n < 0 || n_rows < 0 || width < 0) return 0;
  r2s::Carver cv(nullptr);
  r2s::carve_bwd(cv, n, n_rows, width);
  return static_cast<int64_t>(cv.used);
}

int r2s_embedding_bwd(const void *v_out, int64_t v_out_stride, const void *ids,
                      int32_t ids_are_64, float scale, int32_t type, int64_t n, int64_t n_rows,
                      int64_t width, void *v_table, void *ws, size_t ws_bytes, r2s_stream_t st) {
  using namespace r2s;
  clear_error();
  R2S_RETURN_IF(check_lookup("embedding_bwd", n, n_rows, width, v_out_stride, type, ids));
  if (n_rows == 0 || width == 0) return R2S_OK;
  R2S_REQUIRE((v_out != nullptr || n == 0) && v_table != nullptr,
              "embedding_bwd: null gradient");
  const int64_t need = r2s_embedding_bwd_workspace_bytes(n, n_rows, width);
  if (ws == nullptr || static_cast<int64_t>(ws_bytes) < need) {
    set_error("embedding_bwd: workspace of %zu bytes, %lld required", ws_bytes, (long long)need);
    return R2S_EWORKSPACE;
  }
  Carver cv(ws);
  const BwdSpace s = carve_bwd(cv, n, n_rows, width);
  hipStream_t stream = as_stream(st);
  R2S_RETURN_IF(
      sort_ids(ids, ids_are_64 != 0, n, n_rows, s.order, s.offsets, s.keys, s.sort, stream));
  // Eight vectors to a row where it has them: 300k x 16 bf16 of 3000 rows, forward
  // and back, 45 us with vectors of 4 bytes and 52 with 16, 400k x 3 f32 45 with
  // 4 bytes and 52 with 8.
  const int size = type_size(type);
  int bytes = run_bytes(width, size);
  while (bytes > size && ceil_div(width * size, bytes) < 8) bytes /= 2;
  R2S_BY_TYPE(type, R2S_BY_VECTOR(T, bytes, {
    return (lookup_bwd<T, V>(v_out, v_out_stride, scale, n, n_rows, width, v_table, s, stream));
  }));
  return R2S_OK;
}

}  // extern "C"
