// Rows of a table by id, scaled, and the table's gradient.
//
//   forward   out_i = s T[id_i]: each thread moves one vector (16 bytes where
//             addresses and strides allow).  Ids outside the table give zero
//             rows, so no id reads out of range.
//   backward  dT_v = s sum_{id_i = v} dy_i, without atomics: the positions are
//             sorted by id (stable, binning.hip), the sorted list is cut into
//             chunks of equal length whatever the ids are, and each chunk sums
//             its runs of equal ids in float32.  A run inside one chunk is a
//             finished row; a run that crosses chunk ends leaves one partial
//             row per chunk, and a second kernel adds those in chunk order and
//             writes the rows that no id names as zeros.  Chunks keep the work
//             even when a few ids own almost every position, and fix the order
//             of the sums.
#include "r2s_latent.h"

namespace r2s {
namespace {

constexpr int kThreads = 256;

// ------------------------------------------------------------- forward ---

constexpr int kFwdVectors = 4;  // vectors per thread

// Block b writes vectors [b, b + 1) * kThreads * kFwdVectors of the output,
// row-major.  vpr: vectors per row.
template <typename T, int V, typename I>
__global__ __launch_bounds__(kThreads) void lookup_fwd_kernel(
    const T *__restrict__ table, int64_t stride, const I *__restrict__ ids, float scale,
    int64_t n, int64_t n_rows, uint32_t vpr, T *__restrict__ out) {
  const int64_t total = n * vpr;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (kThreads * kFwdVectors);
  // Row and vector of the block's first one; the rest from there in 32 bits.
  const int64_t row0 = base / vpr;
  const uint32_t vec0 = static_cast<uint32_t>(base - row0 * vpr);
  int64_t id[kFwdVectors];
  uint32_t vec[kFwdVectors];
#pragma unroll
  for (int k = 0; k < kFwdVectors; ++k) {
    const uint32_t q = vec0 + k * kThreads + threadIdx.x;
    const uint32_t r = q / vpr;
    vec[k] = q - r * vpr;
    const int64_t row = row0 + r;
    id[k] = row < n ? static_cast<int64_t>(ids[row]) : -1;
  }
  Pack<T, V> x[kFwdVectors];
#pragma unroll
  for (int k = 0; k < kFwdVectors; ++k) {
    if (id[k] >= 0 && id[k] < n_rows) {
      x[k] = load_pack<T, V>(table + id[k] * stride + static_cast<int64_t>(vec[k]) * V);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) x[k].v[j] = static_cast<T>(0.0f);
    }
  }
#pragma unroll
  for (int k = 0; k < kFwdVectors; ++k) {
    const int64_t at = base + k * kThreads + threadIdx.x;
    if (at < total) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        x[k].v[j] = static_cast<T>(static_cast<float>(x[k].v[j]) * scale);
      store_pack<T, V>(out + at * V, x[k]);
    }
  }
}

// ------------------------------------------------------------ backward ---

constexpr int kChunk = 32;     // sorted positions per chunk
constexpr int kInFlight = 8;   // rows loaded before their first use
constexpr int kLongRow = 64;   // chunks: longer rows are added by a whole block

// The backward's view of the sorted list.
struct Sorted {
  const int32_t *order;    // position of each sorted entry
  const int32_t *offsets;  // [n_rows + 1]; offsets[n_rows]: entries in all
};

// lanes = 2^lane_bits lanes hold one row's columns [c0, c0 + lanes V) and walk
// one chunk; partial [chunks][2][width]: slot 0 the chunk's part of a run that
// began in an earlier chunk, slot 1 its part of one that goes on into the
// next (a run that does both is in slot 0).
template <typename T, int V, typename I>
__global__ __launch_bounds__(kThreads) void lookup_bwd_chunks_kernel(
    const T *__restrict__ v_out, int64_t stride, const I *__restrict__ ids, Sorted list,
    float scale, int64_t n_rows, uint32_t width, uint32_t lane_bits, T *__restrict__ v_table,
    float *__restrict__ partial) {
  const uint32_t col = (blockIdx.y << lane_bits) * V + (threadIdx.x & ((1u << lane_bits) - 1u)) * V;
  const int64_t chunk = (static_cast<int64_t>(blockIdx.x) << (8 - lane_bits)) +
                        (threadIdx.x >> lane_bits);
  const int64_t j0 = chunk * kChunk;
  const int64_t n = list.offsets[n_rows];
  if (j0 >= n || col >= width) return;
  const int64_t j1 = min(j0 + kChunk, n);
  const int64_t before = j0 > 0 ? static_cast<int64_t>(ids[list.order[j0 - 1]]) : -1;
  const int64_t after = j1 < n ? static_cast<int64_t>(ids[list.order[j1]]) : -1;
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.0f;
  int64_t run = static_cast<int64_t>(ids[list.order[j0]]);
  bool first = true;  // the run that began at j0
  auto flush = [&](bool last) {
    if ((first && run == before) || (last && run == after)) {
      const int slot = first && run == before ? 0 : 1;
      float *p = partial + (chunk * 2 + slot) * width + col;
#pragma unroll
      for (int v = 0; v < V; ++v) p[v] = acc[v];
    } else {
      Pack<T, V> r;
#pragma unroll
      for (int v = 0; v < V; ++v) r.v[v] = static_cast<T>(acc[v] * scale);
      store_pack<T, V>(v_table + run * width + col, r);
    }
  };
  for (int64_t j = j0; j < j1; j += kInFlight) {
    int64_t id[kInFlight];
    Pack<T, V> x[kInFlight];
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      const int64_t at = list.order[min(j + k, j1 - 1)];
      id[k] = static_cast<int64_t>(ids[at]);
      x[k] = load_pack<T, V>(v_out + at * stride + col);
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

// Blocks from n_long on: one row per lane group -- zeros without an entry,
// the sum of its parts if it crosses a chunk end, nothing to do otherwise.
// Blocks before: block b looks at the row that holds the first entry of chunk
// (b + 1) kLongRow and adds its parts if it spans more than kLongRow chunks
// and no smaller b sees it.
template <typename T, int V, typename I>
__global__ __launch_bounds__(kThreads) void lookup_bwd_rows_kernel(
    const I *__restrict__ ids, Sorted list, float scale, int64_t n_rows, uint32_t width,
    uint32_t lane_bits, uint32_t n_long, const float *__restrict__ partial,
    T *__restrict__ v_table) {
  const uint32_t lane = threadIdx.x & ((1u << lane_bits) - 1u), group = threadIdx.x >> lane_bits;
  const uint32_t groups = kThreads >> lane_bits;
  const uint32_t col = (blockIdx.y << lane_bits) * V + lane * V;
  const bool inside = col < width;
  __shared__ float sums[kThreads * V];
  int64_t row;
  bool whole = blockIdx.x < n_long;
  if (whole) {
    const int64_t j = (static_cast<int64_t>(blockIdx.x) + 1) * kLongRow * kChunk;
    if (j >= list.offsets[n_rows]) return;
    row = static_cast<int64_t>(ids[list.order[j]]);
  } else {
    row = (static_cast<int64_t>(blockIdx.x) - n_long) * groups + group;
    if (row >= n_rows) return;
  }
  const int64_t o0 = list.offsets[row], o1 = list.offsets[row + 1];
  const int64_t c0 = o0 / kChunk, c1 = o1 > o0 ? (o1 - 1) / kChunk : c0;
  const bool is_long = c1 - c0 > kLongRow;
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.0f;
  if (whole) {
    // Uniform over the block: every thread of a block reads the same row.
    const int64_t smaller = static_cast<int64_t>(blockIdx.x) * kLongRow * kChunk;
    if (!is_long || (blockIdx.x > 0 && o0 <= smaller)) return;
    for (int64_t c = c0 + group; c <= c1; c += groups) {
      if (inside) {
        const float *p = partial + (c * 2 + (c == c0 ? 1 : 0)) * width + col;
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] += p[v];
      }
    }
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
    if (inside && o1 > o0) {
      for (int64_t c = c0; c <= c1; ++c) {
        const float *p = partial + (c * 2 + (c == c0 ? 1 : 0)) * width + col;
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] += p[v];
      }
    }
  }
  if (!inside) return;
  Pack<T, V> r;
#pragma unroll
  for (int v = 0; v < V; ++v) r.v[v] = static_cast<T>(acc[v] * scale);
  store_pack<T, V>(v_table + row * width + col, r);
}

// ---------------------------------------------------------------- host ---

struct BwdSpace {
  int32_t *order, *offsets;
  float *partial;
  char *sort;
};

BwdSpace carve_bwd(Carver &cv, int64_t n, int64_t n_rows, int64_t width) {
  BwdSpace s;
  s.order = cv.take<int32_t>(n);
  s.offsets = cv.take<int32_t>(n_rows + 1);
  s.partial = cv.take<float>(ceil_div(n, kChunk) * 2 * width);
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
  const uint32_t vpr = static_cast<uint32_t>(width / V);
  const int64_t blocks = ceil_div(n * vpr, kThreads * kFwdVectors);
  if (blocks > kInt32Max) {
    set_error("embedding_fwd: output too large");
    return R2S_ERANGE;
  }
  lookup_fwd_kernel<T, V, I><<<dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, stream>>>(
      static_cast<const T *>(table), stride, static_cast<const I *>(ids), scale, n, n_rows, vpr,
      static_cast<T *>(out));
  return check_launch("embedding_fwd");
}

template <typename T, int V, typename I>
int lookup_bwd(const void *v_out, int64_t stride, const void *ids_, float scale, int64_t n,
               int64_t n_rows, int64_t width_, void *v_table_, const BwdSpace &s,
               hipStream_t stream) {
  const I *ids = static_cast<const I *>(ids_);
  T *v_table = static_cast<T *>(v_table_);
  const uint32_t width = static_cast<uint32_t>(width_), vpr = width / V;
  uint32_t bits = 0;
  while (bits < 6 && (1u << bits) < vpr) ++bits;
  const uint32_t slices = static_cast<uint32_t>(ceil_div(vpr, 1 << bits));
  const int64_t groups = kThreads >> bits, chunks = ceil_div(n, kChunk);
  const Sorted list{s.order, s.offsets};
  if (n > 0) {
    lookup_bwd_chunks_kernel<T, V, I>
        <<<dim3(static_cast<uint32_t>(ceil_div(chunks, groups)), slices), dim3(kThreads), 0,
           stream>>>(static_cast<const T *>(v_out), stride, ids, list, scale, n_rows, width, bits,
                     v_table, s.partial);
    R2S_RETURN_IF(check_launch("embedding_bwd"));
  }
  const int64_t n_long = chunks > 0 ? (chunks - 1) / kLongRow : 0;
  lookup_bwd_rows_kernel<T, V, I>
      <<<dim3(static_cast<uint32_t>(n_long + ceil_div(n_rows, groups)), slices), dim3(kThreads),
         0, stream>>>(ids, list, scale, n_rows, width, bits, static_cast<uint32_t>(n_long),
                      s.partial, v_table);
  return check_launch("embedding_bwd rows");
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
  const uint64_t size = type_size(type);
  const int bytes = vector_bytes({address(table), address(out), table_stride * size, width * size},
                                 static_cast<int>(size));
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
  R2S_RETURN_IF(sort_ids(ids, ids_are_64 != 0, n, n_rows, s.order, s.offsets, s.sort, stream));
  const uint64_t size = type_size(type);
  const int bytes = vector_bytes({address(v_out), address(v_table), v_out_stride * size,
                                  width * size},
                                 static_cast<int>(size));
  R2S_BY_TYPE(type, R2S_BY_VECTOR(T, bytes, {
    return ids_are_64 ? (lookup_bwd<T, V, int64_t>(v_out, v_out_stride, ids, scale, n, n_rows,
                                                   width, v_table, s, stream))
                      : (lookup_bwd<T, V, int32_t>(v_out, v_out_stride, ids, scale, n, n_rows,
                                                   width, v_table, s, stream));
  }));
  return R2S_OK;
}

}  // extern "C"
