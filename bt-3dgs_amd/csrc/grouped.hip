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
// Every product is a 64 x 64 tile per block of four waves on the matrix cores,
// operands staged in LDS with the summed index innermost; sums are float32.
// dW sums over rows: its blocks take a fixed number of rows of one group each
// and leave float32 parts, which a second kernel adds in row order.
#include "r2s_latent.h"

namespace r2s {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64;        // rows and columns of a block's tile
constexpr int kSlabBytes = 128;  // of the summed index per stage
constexpr int kPitch = kSlabBytes + 16;

using f32x4 = __attribute__((ext_vector_type(4))) float;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;

// acc += A B over the 16 bytes per lane of the summed index (which elements
// they are does not matter, as long as both operands hold the same).
template <typename T>
__device__ __forceinline__ void multiply(const void *a, const void *b, f32x4 &acc) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 x = *static_cast<const f32x4 *>(a), y = *static_cast<const f32x4 *>(b);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], acc, 0, 0, 0);
  } else if constexpr (std::is_same<T, bf16_t>::value) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*static_cast<const bf16x8 *>(a),
                                                  *static_cast<const bf16x8 *>(b), acc, 0, 0, 0);
  } else {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(*static_cast<const f16x8 *>(a),
                                                 *static_cast<const f16x8 *>(b), acc, 0, 0, 0);
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

// Part `slot` of the groups cut into parts of `per` rows each: its group and
// rows [r0, r1).  With `rest` the rows past the last group follow as group
// `count`.  False past the last part.  Called by whole waves.
__device__ __forceinline__ bool find_part(const Groups &g, bool rest, uint32_t per, uint32_t slot,
                                          int32_t &group, int64_t &r0, int64_t &r1) {
  uint32_t before = 0;
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
    const uint64_t past = ballot(end > slot);
    if (past != 0) {
      const uint32_t src = static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(past))) - 1u;
      group = static_cast<int32_t>(readlane_u32(static_cast<uint32_t>(e), src));
      const uint32_t first = readlane_u32(end - parts, src);
      r0 = readlane_i64(lo, src) + static_cast<int64_t>(slot - first) * per;
      r1 = min(readlane_i64(hi, src), r0 + per);
      return true;
    }
    before = readlane_u32(end, 63);
  }
  return false;
}

// ------------------------------------------------------------- staging ---

// Stages [kTile][slab] of an operand whose summed index is innermost in
// memory: element (r, c) at base + row(r) * stride + c0 + c; rows < 0 and
// c0 + c >= c_end are zero.
template <typename T, bool kVec, typename Row>
__device__ __forceinline__ void stage_along(char *lds, const T *base, int64_t stride, Row row,
                                            int64_t c0, int64_t c_end) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  constexpr int kChunks = kTile * kSlabBytes / 16 / kThreads;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int q = threadIdx.x + i * kThreads, r = q / (kSlabBytes / 16), s = q % (kSlabBytes / 16);
    const int64_t at = row(r), c = c0 + s * kPer;
    Pack<T, kPer> x;
    if (kVec && at >= 0 && c + kPer <= c_end) {
      x = load_pack<T, kPer>(base + at * stride + c);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        x.v[j] = at >= 0 && c + j < c_end ? base[at * stride + c + j] : static_cast<T>(0.0f);
    }
    *reinterpret_cast<Pack<T, kPer> *>(lds + r * kPitch + s * 16) = x;
  }
}

// The same of an operand whose tile rows are innermost in memory: element
// (r, c) at base + row(c) * stride + r0 + r; r0 + r >= r_end is zero.
template <typename T, bool kVec, typename Row>
__device__ __forceinline__ void stage_across(char *lds, const T *base, int64_t stride, Row row,
                                             int64_t r0, int64_t r_end) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  constexpr int kChunks = kTile * kSlabBytes / 16 / kThreads;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int q = threadIdx.x + i * kThreads, c = q / (kTile / kPer), s = q % (kTile / kPer);
    const int64_t at = row(c), r = r0 + s * kPer;
    Pack<T, kPer> x;
    if (kVec && at >= 0 && r + kPer <= r_end) {
      x = load_pack<T, kPer>(base + at * stride + r);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        x.v[j] = at >= 0 && r + j < r_end ? base[at * stride + r + j] : static_cast<T>(0.0f);
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      *reinterpret_cast<T *>(lds + (s * kPer + j) * kPitch + c * sizeof(T)) = x.v[j];
  }
}

// The staged slab's products: wave (wm, wn) of the 2 x 2 has 32 x 32.
template <typename T>
__device__ __forceinline__ void multiply_slab(const char *a, const char *b, f32x4 (&acc)[2][2]) {
  const int lane = threadIdx.x % 64, wm = threadIdx.x / 128, wn = (threadIdx.x / 64) % 2;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int at = half * 64 + lane / 16 * 16;
    const char *pa = a + (wm * 32 + lane % 16) * kPitch + at;
    const char *pb = b + (wn * 32 + lane % 16) * kPitch + at;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        multiply<T>(pa + i * 16 * kPitch, pb + j * 16 * kPitch, acc[i][j]);
  }
}

// store(row, column, value) for each element of the block's tile.
template <typename Store>
__device__ __forceinline__ void store_tile(const f32x4 (&acc)[2][2], Store store) {
  const int lane = threadIdx.x % 64, wm = threadIdx.x / 128, wn = (threadIdx.x / 64) % 2;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        store(wm * 32 + i * 16 + lane / 16 * 4 + k, wn * 32 + j * 16 + lane % 16, acc[i][j][k]);
}

// ------------------------------------------------------------- kernels ---

// Rows times weights: out[r][j] = sum_c in[r][c] w(c, j), the forward
// (weight [m, k], summed over k) or with kBack the input's gradient (summed
// over m).
template <typename T, bool kBack, bool kVec>
__global__ __launch_bounds__(kThreads) void rows_kernel(const T *__restrict__ in, int64_t stride,
                                                        const T *__restrict__ weight,
                                                        const T *__restrict__ bias, Groups g,
                                                        const int32_t *__restrict__ rows,
                                                        int64_t k, int64_t m,
                                                        T *__restrict__ out) {
  __shared__ __attribute__((aligned(16))) char s_a[kTile * kPitch], s_b[kTile * kPitch];
  __shared__ int64_t s_row[kTile];
  constexpr int kSlab = kSlabBytes / static_cast<int>(sizeof(T));
  const int64_t inner = kBack ? m : k, outer = kBack ? k : m;
  int32_t e;
  int64_t r0, r1;
  if (!find_part(g, true, kTile, blockIdx.x, e, r0, r1)) return;
  if (threadIdx.x < kTile) {
    const int64_t i = r0 + threadIdx.x;
    int64_t r = -1;
    if (i < r1) {
      r = rows != nullptr ? rows[i] : i;
      if (r >= g.n) r = -1;
    }
    s_row[threadIdx.x] = r;
  }
  __syncthreads();
  const int64_t j0 = static_cast<int64_t>(blockIdx.y) * kTile;
  f32x4 acc[2][2] = {};
  if (e < g.count) {
    const T *w = weight + static_cast<int64_t>(e) * m * k;
    for (int64_t c0 = 0; c0 < inner; c0 += kSlab) {
      stage_along<T, kVec>(s_a, in, stride, [&](int r) { return s_row[r]; }, c0, inner);
      if constexpr (kBack)
        stage_across<T, kVec>(
            s_b, w, k, [&](int c) { return c0 + c < m ? c0 + c : int64_t{-1}; }, j0, k);
      else
        stage_along<T, kVec>(
            s_b, w, k, [&](int r) { return j0 + r < m ? j0 + r : int64_t{-1}; }, c0, k);
      __syncthreads();
      multiply_slab<T>(s_a, s_b, acc);
      __syncthreads();
    }
  }
  store_tile(acc, [&](int r, int c, float v) {
    const int64_t at = s_row[r], j = j0 + c;
    if (at < 0 || j >= outer) return;
    if (!kBack && bias != nullptr && e < g.count)
      v += static_cast<float>(bias[static_cast<int64_t>(e) * m + j]);
    out[at * outer + j] = static_cast<T>(v);
  });
}

// Parts of dW (and db): part s of `per` rows of one group, tile (y, z) of
// [m, k], into parts [slots][m][k] and bias_parts [slots][m] (may be null).
template <typename T, bool kVec>
__global__ __launch_bounds__(kThreads) void weights_kernel(
    const T *__restrict__ x, int64_t x_stride, const T *__restrict__ v_y, int64_t v_stride,
    Groups g, const int32_t *__restrict__ rows, int64_t k, int64_t m, uint32_t per,
    float *__restrict__ parts, float *__restrict__ bias_parts) {
  __shared__ __attribute__((aligned(16))) char s_a[kTile * kPitch], s_b[kTile * kPitch];
  constexpr int kSlab = kSlabBytes / static_cast<int>(sizeof(T));
  __shared__ int64_t s_row[kSlab];
  int32_t e;
  int64_t r0, r1;
  if (!find_part(g, false, per, blockIdx.x, e, r0, r1)) return;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kTile;
  const int64_t k0 = static_cast<int64_t>(blockIdx.z) * kTile;
  f32x4 acc[2][2] = {};
  float bias_sum = 0.0f;
  for (int64_t c0 = r0; c0 < r1; c0 += kSlab) {
    if (threadIdx.x < kSlab) {
      const int64_t i = c0 + threadIdx.x;
      int64_t r = -1;
      if (i < r1) {
        r = rows != nullptr ? rows[i] : i;
        if (r >= g.n) r = -1;
      }
      s_row[threadIdx.x] = r;
    }
    __syncthreads();
    stage_across<T, kVec>(s_a, v_y, v_stride, [&](int c) { return s_row[c]; }, m0, m);
    stage_across<T, kVec>(s_b, x, x_stride, [&](int c) { return s_row[c]; }, k0, k);
    __syncthreads();
    multiply_slab<T>(s_a, s_b, acc);
    if (bias_parts != nullptr && blockIdx.z == 0 && threadIdx.x < kTile) {
      for (int c = 0; c < kSlab; ++c)
        bias_sum += static_cast<float>(
            *reinterpret_cast<const T *>(s_a + threadIdx.x * kPitch + c * sizeof(T)));
    }
    __syncthreads();
  }
  float *p = parts + static_cast<int64_t>(blockIdx.x) * m * k;
  store_tile(acc, [&](int r, int c, float v) {
    if (m0 + r < m && k0 + c < k) p[(m0 + r) * k + k0 + c] = v;
  });
  if (bias_parts != nullptr && blockIdx.z == 0 && threadIdx.x < kTile && m0 + threadIdx.x < m)
    bias_parts[static_cast<int64_t>(blockIdx.x) * m + m0 + threadIdx.x] = bias_sum;
}

// out[e][i] = the sum of group e's parts, in row order.
template <typename T>
__global__ __launch_bounds__(kThreads) void add_parts_kernel(const float *__restrict__ parts,
                                                             Groups g, uint32_t per,
                                                             uint32_t slots, int64_t size,
                                                             T *__restrict__ out) {
  const int32_t e = static_cast<int32_t>(blockIdx.y);
  uint32_t before = 0, mine = 0;
  for (int32_t e0 = 0; e0 <= e; e0 += 64) {
    const int32_t q = e0 + static_cast<int32_t>(lane_id());
    uint32_t n = 0;
    if (q <= e) {
      const int64_t rows = g.bound(q + 1) - g.bound(q);
      n = rows > 0 ? static_cast<uint32_t>((rows + per - 1) / per) : 0u;
    }
    const uint32_t end = before + wave_inclusive_scan(n);
    mine = readlane_u32(n, static_cast<uint32_t>(min(e - e0, 63)));
    before = readlane_u32(end, 63);
  }
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= size) return;
  // Offsets that do not ascend could name more parts than there are.
  const uint32_t first = min(before - mine, slots);
  mine = min(mine, slots - first);
  const float *p = parts + static_cast<int64_t>(first) * size + i;
  float sum = 0.0f;
#pragma unroll 4
  for (uint32_t s = 0; s < mine; ++s) sum += p[static_cast<int64_t>(s) * size];
  out[static_cast<int64_t>(e) * size + i] = static_cast<T>(sum);
}

// ---------------------------------------------------------------- host ---

uint32_t rows_per_part(int64_t k, int64_t m) {
  return ceil_div(k, kTile) * ceil_div(m, kTile) >= 64 ? 4096 : 1024;
}

// Blocks of the weights' gradient along the rows, at most.
int64_t part_slots(int64_t n, int64_t k, int64_t m, int64_t groups) {
  return ceil_div(n, rows_per_part(k, m)) + groups;
}

struct GradSpace {
  float *parts, *bias_parts;
};
GradSpace carve_grad(Carver &cv, int64_t n, int64_t k, int64_t m, int64_t groups) {
  const int64_t slots = part_slots(n, k, m, groups);
  GradSpace s;
  s.parts = cv.take<float>(slots * m * k);
  s.bias_parts = cv.take<float>(slots * m);
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

template <typename T, bool kBack>
int rows_product(const void *in, int64_t stride, const void *weight, const void *bias, Groups g,
                 const int32_t *rows, int64_t k, int64_t m, void *out, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(ceil_div(g.n, kTile) + g.count + 1),
                  static_cast<uint32_t>(ceil_div(kBack ? k : m, kTile)));
  const bool vec = address(in) % 16 == 0 && address(weight) % 16 == 0 &&
                   stride * sizeof(T) % 16 == 0 && k * sizeof(T) % 16 == 0;
  const T *ti = static_cast<const T *>(in), *tw = static_cast<const T *>(weight);
  const T *tb = static_cast<const T *>(bias);
  if (vec)
    rows_kernel<T, kBack, true><<<grid, dim3(kThreads), 0, stream>>>(ti, stride, tw, tb, g, rows,
                                                                     k, m, static_cast<T *>(out));
  else
    rows_kernel<T, kBack, false><<<grid, dim3(kThreads), 0, stream>>>(ti, stride, tw, tb, g, rows,
                                                                      k, m, static_cast<T *>(out));
  return check_launch("grouped_matmul");
}

template <typename T>
int weights_product(const void *x, int64_t x_stride, const void *v_y, int64_t v_stride, Groups g,
                    const int32_t *rows, int64_t k, int64_t m, void *v_weight, void *v_bias,
                    const GradSpace &s, hipStream_t stream) {
  const uint32_t per = rows_per_part(k, m);
  const uint32_t slots = static_cast<uint32_t>(part_slots(g.n, k, m, g.count));
  float *bias_parts = v_bias != nullptr ? s.bias_parts : nullptr;
  if (g.n > 0) {
    const dim3 grid(slots,
                    static_cast<uint32_t>(ceil_div(m, kTile)),
                    static_cast<uint32_t>(max(ceil_div(k, kTile), int64_t{1})));
    const bool vec = address(x) % 16 == 0 && address(v_y) % 16 == 0 &&
                     x_stride * sizeof(T) % 16 == 0 && v_stride * sizeof(T) % 16 == 0;
    const T *tx = static_cast<const T *>(x), *tv = static_cast<const T *>(v_y);
    if (vec)
      weights_kernel<T, true><<<grid, dim3(kThreads), 0, stream>>>(tx, x_stride, tv, v_stride, g,
                                                                   rows, k, m, per, s.parts,
                                                                   bias_parts);
    else
      weights_kernel<T, false><<<grid, dim3(kThreads), 0, stream>>>(tx, x_stride, tv, v_stride, g,
                                                                    rows, k, m, per, s.parts,
                                                                    bias_parts);
    R2S_RETURN_IF(check_launch("grouped_matmul_bwd weights"));
  }
  if (v_weight != nullptr && m * k > 0) {
    add_parts_kernel<T><<<dim3(static_cast<uint32_t>(ceil_div(m * k, kThreads)), g.count),
                          dim3(kThreads), 0, stream>>>(s.parts, g, per, slots, m * k,
                                                       static_cast<T *>(v_weight));
    R2S_RETURN_IF(check_launch("grouped_matmul_bwd weights"));
  }
  if (v_bias != nullptr) {
    add_parts_kernel<T><<<dim3(static_cast<uint32_t>(ceil_div(m, kThreads)), g.count),
                          dim3(kThreads), 0, stream>>>(s.bias_parts, g, per, slots, m,
                                                       static_cast<T *>(v_bias));
    R2S_RETURN_IF(check_launch("grouped_matmul_bwd bias"));
  }
  return R2S_OK;
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

int64_t r2s_grouped_matmul_bwd_workspace_bytes(int64_t n, int64_t k, int64_t m, int64_t groups) {
  if (n < 0 || k < 0 || m < 0 || groups < 0) return 0;
  r2s::Carver cv(nullptr);
  r2s::carve_grad(cv, n, k, m, groups);
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
  const int64_t need = r2s_grouped_matmul_bwd_workspace_bytes(n, k, m, groups);
  if (ws == nullptr || static_cast<int64_t>(ws_bytes) < need) {
    set_error("grouped_matmul_bwd: workspace of %zu bytes, %lld required", ws_bytes,
              (long long)need);
    return R2S_EWORKSPACE;
  }
  Carver cv(ws);
  const GradSpace s = carve_grad(cv, n, k, m, groups);
  R2S_BY_TYPE(type, return (weights_product<T>(x, x_stride, v_y, v_y_stride, g, rows, k, m,
                                               v_weight, v_bias, s, stream)));
  return R2S_OK;
}

}  // extern "C"
