// The norms around a block, with its gate and the residual scale between them:
//
//   h = norm(f) w1   (f itself without w1),
//   y = x + s sigmoid(g) h,
//   u = norm(y) w2,  norm(z) = (z - c) / sqrt(mean((z - c)^2) + eps),
//
// c the row's mean or 0.  With m(a) the row's mean of a, the gradient of
// v = norm(z) w is r (v' - n m(v' n) - c'), v' = v w, n = norm(z), r its factor and
// c' = m(v') where c is the mean, else 0.
//
// A row is held in registers by 8 to 512 lanes, 16 bytes of each input a lane (more
// only where a row has over 512 such pieces: two to each of 64 lanes took 503 us where
// one to each of 128 took 216, 32k x 1024 bfloat16 both ways), so each input is read
// once and each output written once, and the sums of squares are of differences from
// the mean that was found first.  The backward makes the
// forward's values again from its inputs, which costs no bytes.  Weights' gradients
// are sums over rows: a lane group adds its rows, a block its groups, and a second
// kernel the blocks, always in the same order.  Bound by the bytes.
#include <algorithm>

#include "r2s_latent.h"

namespace r2s {
namespace {

constexpr int kNormMost = 8192;   // channels

enum : int { kNoGate = 0, kRowGate = 1, kChannelGate = 2 };

struct NormInput {
  const void *p;
  int64_t stride;
};

struct NormArgs {
  NormInput x, update, gate, v_y, v_u;
  const void *w1, *w2;
  void *y, *u;                        // forward
  void *v_x, *v_update, *v_gate;      // backward (v_gate: of every row)
  float *parts;                       // [blocks][3][d]: v_w1, v_w2, v_gate of all rows
  int64_t n;
  int32_t d, gate_kind, centered;
  int32_t want_w1, want_w2, want_gate;  // sums over rows
  float scale, eps;
};

template <typename T, int V>
struct __attribute__((packed)) Loose {
  T v[V];
};

// `count` of V elements at any element, zeros for the others.
template <typename T, int V>
__device__ __forceinline__ Loose<T, V> load_row(const T *p, int count) {
  if (count >= V) return *reinterpret_cast<const Loose<T, V> *>(p);
  Loose<T, V> x;
#pragma unroll
  for (int i = 0; i < V; ++i) x.v[i] = i < count ? p[i] : static_cast<T>(0.0f);
  return x;
}
template <typename T, int V>
__device__ __forceinline__ void store_row(T *p, int count, const Loose<T, V> &x) {
  if (count >= V) {
    *reinterpret_cast<Loose<T, V> *>(p) = x;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < count) p[i] = x.v[i];
  }
}

// sigmoid(g) and 1 - sigmoid(g), each within a few units of float32's last place: the
// hardware's exponential and reciprocal are within one, and what rounding the
// exponential's argument in units of log 2 leaves is put back.  Below 2^-126 it is 0.
__device__ __forceinline__ float2 sigmoids(float g) {
  constexpr float kLog2e = 1.44269502162933349609f, kRest = 1.92596299e-8f;  // of log2(e)
  const float x = -fabsf(g), t = x * kLog2e;
  const float left = fmaf(x, kRest, fmaf(x, kLog2e, -t));
  const float near = __builtin_amdgcn_exp2f(t);
  // An infinite x leaves a NaN beside its exponential of 0.
  const float e = near == 0.0f ? 0.0f : fmaf(near, left * 0.693147180559945f, near);
  const float big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
  return g >= 0.0f ? make_float2(big, small) : make_float2(small, big);
}

// The sum over the 2^bits lanes (aligned, bits >= 3) that hold a row's part of a wave:
// lanes 1, 2, 4 and 8 apart by moves within rows of 16 lanes (by then whole quads and
// halves agree, so mirrors do), 16 and 32 by swaps of such rows.
__device__ __forceinline__ float lanes_sum(float a, int bits) {
  a += dpp_take<0xB1, 0xf>(a);   // quad_perm 1 0 3 2
  a += dpp_take<0x4E, 0xf>(a);   // quad_perm 2 3 0 1
  a += dpp_take<0x141, 0xf>(a);  // row_half_mirror
  if (bits > 3) a += dpp_take<0x140, 0xf>(a);  // row_mirror
  if (bits > 4) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(a), false,
                                                    false);
    a = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (bits > 5) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(a), false,
                                                    false);
    a = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return a;
}

// The lanes of a row: 2^bits of a wave, or (kWide, bits > 6) of several waves.
template <bool kWide, int kThreads>
struct Lanes {
  static constexpr int kWaves = kThreads / 64;
  int bits, lane;
  float2 *s_sums;  // [2][kWaves], kWide
  int turn = 0;
  __device__ __forceinline__ Lanes(int b, float2 *sums) : bits(b), s_sums(sums) {
    lane = static_cast<int>(threadIdx.x) & ((1 << bits) - 1);
  }
  __device__ __forceinline__ float2 sum(float a, float b) {
    a = lanes_sum(a, kWide ? 6 : bits);
    b = lanes_sum(b, kWide ? 6 : bits);
    return across(a, b);
  }
  __device__ __forceinline__ float sum(float a) {
    a = lanes_sum(a, kWide ? 6 : bits);
    return across(a, 0.0f).x;
  }

 private:
  // The sums of all the row's waves, the same bits in each.
  __device__ __forceinline__ float2 across(float a, float b) {
    float2 total = make_float2(a, b);
    if constexpr (kWide) {
      float2 *at = s_sums + turn * kWaves;
      turn ^= 1;  // the sums before the last ones have been read by all
      if (lane_id() == 0) at[wave_index()] = make_float2(a, b);
      __syncthreads();
      const int waves = 1 << (bits - 6), first = static_cast<int>(wave_index()) & ~(waves - 1);
      total = at[first];
      for (int i = 1; i < waves; ++i) {
        total.x += at[first + i].x;
        total.y += at[first + i].y;
      }
    }
    return total;
  }
};

// A lane's share of a row: E vectors of V elements, 2^bits V apart.
template <typename T, int E>
struct Row {
  static constexpr int V = 16 / static_cast<int>(sizeof(T));
  float v[E][V];
};

// Where a lane's vectors are.  Rows are read by whole vectors alone, so that no load
// waits at the end of a branch for the one before it (32k x 1024 bfloat16, backward:
// 131 us, with a branch to each 154): the last vector of a row that ends inside it is
// read from earlier elements on and moved (kTail), and vectors behind the row's end
// are another's that count for nothing.  Such ends of float32 rows, of three elements
// at most, are cheaper read by elements (300k x 45, backward: 71 us, moved 94), and so
// are rows narrower than a vector (kElements).
enum : int { kWhole = 0, kTail = 1, kElements = 2 };
template <typename T, int E, bool kWide, int kThreads, int kEnd>
struct RowOf {
  static constexpr int V = Row<T, E>::V;
  int first[E], count[E];
  int start[E];  // where a vector is read from
  float share;   // 1 / d
  __device__ __forceinline__ RowOf(const Lanes<kWide, kThreads> &lanes, int d) : share(1.0f / d) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      first[e] = ((e << lanes.bits) + lanes.lane) * V;
      count[e] = max(0, min(V, d - first[e]));
      start[e] = kEnd == kElements ? first[e] : min(first[e], d - V);
    }
  }
  __device__ __forceinline__ void load(const NormInput &in, int64_t row,
                                       Loose<T, V> (&raw)[E]) const {
    const T *p = static_cast<const T *>(in.p) + row * in.stride;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (kEnd == kElements) {
        raw[e] = load_row<T, V>(p + first[e], count[e]);
      } else {
        raw[e] = *reinterpret_cast<const Loose<T, V> *>(p + start[e]);
      }
    }
  }
  // A loaded row's own elements, and zeros past its end.
  __device__ __forceinline__ void settle(Loose<T, V> (&raw)[E]) const {
    if constexpr (kEnd == kElements) return;
    using Words = __attribute__((ext_vector_type(4))) uint32_t;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      Words x = __builtin_bit_cast(Words, raw[e]);
      if constexpr (kEnd == kTail) {
        static_assert(sizeof(T) == 2, "two elements to a word");
        const int back = first[e] - start[e];  // of the row's last vector
#pragma unroll
        for (int words = 2; words > 0; words /= 2)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            x[j] = (back & (2 * words)) != 0 ? (j + words < 4 ? x[j + words] : 0u) : x[j];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[j] = (back & 1) != 0 ? x[j] >> 16 | (j < 3 ? x[j + 1] << 16 : 0u) : x[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = count[e] > 0 ? x[j] : 0u;
      raw[e] = __builtin_bit_cast(Loose<T, V>, x);
    }
  }
  // A weight (ones without one), zeros past the row's end.
  __device__ __forceinline__ void load_weight(const void *w, Row<T, E> &out) const {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const Loose<T, V> raw =
          load_row<T, V>(static_cast<const T *>(w) + first[e], w != nullptr ? count[e] : 0);
#pragma unroll
      for (int i = 0; i < V; ++i)
        out.v[e][i] = w != nullptr ? static_cast<float>(raw.v[i]) : (i < count[e] ? 1.0f : 0.0f);
    }
  }
  __device__ __forceinline__ void store(void *out, int64_t row, int d, const Row<T, E> &x) const {
    T *p = static_cast<T *>(out) + row * d;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      Loose<T, V> raw;
#pragma unroll
      for (int i = 0; i < V; ++i) raw.v[i] = static_cast<T>(x.v[e][i]);
      store_row<T, V>(p + first[e], count[e], raw);
    }
  }
  // x <- norm(x); returns the factor.
  __device__ __forceinline__ float norm(Lanes<kWide, kThreads> &lanes, bool centered, float eps,
                                        Row<T, E> &x) const {
    if (centered) {
      float total = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < V; ++i) total += x.v[e][i];
      const float mean = lanes.sum(total) * share;
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < V; ++i) x.v[e][i] = i < count[e] ? x.v[e][i] - mean : 0.0f;
    }
    float total = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < V; ++i) total = fmaf(x.v[e][i], x.v[e][i], total);
    const float factor = 1.0f / sqrtf(fmaf(lanes.sum(total), share, eps));
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < V; ++i) x.v[e][i] *= factor;
    return factor;
  }
};

template <typename T, int E>
__device__ __forceinline__ void widen(const Loose<T, Row<T, E>::V> (&raw)[E], Row<T, E> &x) {
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int i = 0; i < Row<T, E>::V; ++i) x.v[e][i] = static_cast<float>(raw[e].v[i]);
}

// 32k x 1024 bfloat16 with a gate of every row: 335 MB in 70 to 73 us (4.6 to 4.8 TB/s);
// 300k x 45 float32 39 to 42 us (5.2 to 5.5 TB/s); 4k x 64 float32 4 us, the launch's
// own.  Bound by the bytes.
template <typename T, int E, bool kWide, int kThreads, int kGate, int kEnd>
__global__ __launch_bounds__(kThreads) void residual_norm_fwd_kernel(NormArgs a, int bits) {
  __shared__ float2 s_sums[2 * (kThreads / 64)];
  constexpr int V = Row<T, E>::V;
  Lanes<kWide, kThreads> lanes(bits, s_sums);
  const RowOf<T, E, kWide, kThreads, kEnd> at(lanes, a.d);
  Row<T, E> w1, w2, all;
  at.load_weight(a.w1, w1);
  at.load_weight(a.w2, w2);
  if constexpr (kGate == kChannelGate) {
    at.load_weight(a.gate.p, all);
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < V; ++i) all.v[e][i] = sigmoids(all.v[e][i]).x;
  }
  const int64_t groups = static_cast<int64_t>(gridDim.x) * (kThreads >> bits);
  int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads >> bits) + (threadIdx.x >> bits);
  // A wave's groups stop together, and with kWide a block's: they add up together.
  const int64_t group0 = row - (threadIdx.x >> bits) + (kWide ? 0 : (threadIdx.x & ~63) >> bits);
  for (int64_t lead = group0; lead < a.n; lead += groups, row += groups) {
    const bool some = row < a.n;
    const int64_t r = some ? row : lead;
    Loose<T, V> rx[E], rf[E], rg[E];
    at.load(a.x, r, rx);
    if (a.update.p != nullptr) at.load(a.update, r, rf);
    if constexpr (kGate == kRowGate) at.load(a.gate, r, rg);
    at.settle(rx);
    if (a.update.p != nullptr) at.settle(rf);
    if constexpr (kGate == kRowGate) at.settle(rg);
    Row<T, E> y;
    widen<T, E>(rx, y);
    if (a.update.p != nullptr) {
      Row<T, E> h;
      widen<T, E>(rf, h);
      if (a.w1 != nullptr) at.norm(lanes, a.centered != 0, a.eps, h);
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float s = a.scale;
          if constexpr (kGate == kRowGate) s *= sigmoids(static_cast<float>(rg[e].v[i])).x;
          if constexpr (kGate == kChannelGate) s *= all.v[e][i];
          y.v[e][i] = fmaf(s, h.v[e][i] * w1.v[e][i], y.v[e][i]);
        }
      if (some) at.store(a.y, r, a.d, y);
    }
    if (a.u != nullptr) {
      at.norm(lanes, a.centered != 0, a.eps, y);
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < V; ++i) y.v[e][i] *= w2.v[e][i];
      if (some) at.store(a.u, r, a.d, y);
    }
  }
}

// A block's sum of its groups' `sums`, into its part.
template <typename T, int E, bool kWide, int kThreads, int kEnd>
__device__ __forceinline__ void store_part(const RowOf<T, E, kWide, kThreads, kEnd> &at, int bits, int d,
                                           const Row<T, E> &sums, float *s_row, float *part) {
  constexpr int V = Row<T, E>::V;
  const int groups = kThreads >> bits;
  float *mine = groups > 1 ? s_row + (threadIdx.x >> bits) * d : part;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < at.count[e]) mine[at.first[e] + i] = sums.v[e][i];
  if (groups == 1) return;
  __syncthreads();
  for (int c = threadIdx.x; c < d; c += kThreads) {
    float total = 0.0f;
    for (int g = 0; g < groups; ++g) total += s_row[g * d + c];
    part[c] = total;
  }
}

// 32k x 1024 bfloat16 with a gate of every row: 537 MB in 117 to 131 us (4.1 to 4.6
// TB/s); 300k x 45 float32 67 to 74 us (4.4 to 4.8 TB/s).  float32 rows of more than 4096
// channels spill six registers, which the bytes cover (4096 x 8192: 245 us, as 8192 x
// 4096).  Between a row's loads and its stores lie
// four sums over its lanes in turn; with 16-bit rows' eight elements to a lane three
// waves of a SIMD are what the registers hold to cover them (eight waves of four
// elements: 234 us against 154).
template <typename T, int E, bool kWide, int kThreads, int kGate, int kEnd>
__global__ __launch_bounds__(kThreads, E > 1 ? 2 : sizeof(T) == 2 ? 3 : 4) void
residual_norm_bwd_kernel(NormArgs a, int bits) {
  __shared__ float2 s_sums[2 * (kThreads / 64)];
  extern __shared__ float s_row[];  // [groups][d], of several groups
  constexpr int V = Row<T, E>::V;
  Lanes<kWide, kThreads> lanes(bits, s_sums);
  const RowOf<T, E, kWide, kThreads, kEnd> at(lanes, a.d);
  const bool centered = a.centered != 0, update = a.update.p != nullptr;
  Row<T, E> w1, w2, all, v_w1{}, v_w2{}, v_all{};
  at.load_weight(a.w1, w1);
  at.load_weight(a.w2, w2);
  if constexpr (kGate == kChannelGate) at.load_weight(a.gate.p, all);
  const int64_t groups = static_cast<int64_t>(gridDim.x) * (kThreads >> bits);
  int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads >> bits) + (threadIdx.x >> bits);
  const int64_t group0 = row - (threadIdx.x >> bits) + (kWide ? 0 : (threadIdx.x & ~63) >> bits);
  for (int64_t lead = group0; lead < a.n; lead += groups, row += groups) {
    const bool some = row < a.n;
    const int64_t r = some ? row : lead;
    Loose<T, V> rx[E], rf[E], rg[E], ry[E], ru[E];
    at.load(a.x, r, rx);
    if (update) at.load(a.update, r, rf);
    if constexpr (kGate == kRowGate) at.load(a.gate, r, rg);
    if (a.v_u.p != nullptr) at.load(a.v_u, r, ru);
    if (a.v_y.p != nullptr) at.load(a.v_y, r, ry);
    at.settle(rx);
    if (update) at.settle(rf);
    if constexpr (kGate == kRowGate) at.settle(rg);
    if (a.v_u.p != nullptr) at.settle(ru);
    if (a.v_y.p != nullptr) at.settle(ry);
    Row<T, E> z, h;
    widen<T, E>(rx, z);
    float h_factor = 1.0f;
    // The gate, and its derivative's factor.
    Row<T, E> up, slope;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float2 g = make_float2(1.0f, 0.0f);
        if constexpr (kGate == kChannelGate) g = sigmoids(all.v[e][i]);
        if constexpr (kGate == kRowGate) g = sigmoids(static_cast<float>(rg[e].v[i]));
        up.v[e][i] = a.scale * g.x;
        slope.v[e][i] = g.y;
      }
    if (update) {
      widen<T, E>(rf, h);
      if (a.w1 != nullptr) h_factor = at.norm(lanes, centered, a.eps, h);
    }
    Row<T, E> v;  // the gradient of y
    if (a.v_y.p != nullptr) {
      widen<T, E>(ry, v);
    } else {
      v = Row<T, E>{};
    }
    if (a.v_u.p != nullptr) {
      if (update) {
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
          for (int i = 0; i < V; ++i)
            z.v[e][i] = fmaf(up.v[e][i], h.v[e][i] * w1.v[e][i], z.v[e][i]);
      }
      const float z_factor = at.norm(lanes, centered, a.eps, z);
      float along = 0.0f, total = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float t = static_cast<float>(ru[e].v[i]) * w2.v[e][i];
          along = fmaf(t, z.v[e][i], along);
          total += t;
        }
      float2 mean = lanes.sum(along, total);
      mean.x *= at.share;
      mean.y *= centered ? at.share : 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float vu = static_cast<float>(ru[e].v[i]), t = vu * w2.v[e][i];
          const float inner = centered ? t - mean.y : t;
          v.v[e][i] = fmaf(z_factor, fmaf(-z.v[e][i], mean.x, inner), v.v[e][i]);
          if (some) v_w2.v[e][i] = fmaf(vu, z.v[e][i], v_w2.v[e][i]);
        }
    }
    if (some && a.v_x != nullptr) at.store(a.v_x, r, a.d, v);
    if (!update) continue;
    // z becomes the gate's gradient, v that of h w1.
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v.v[e][i] *= up.v[e][i];
        z.v[e][i] = v.v[e][i] * slope.v[e][i] * (h.v[e][i] * w1.v[e][i]);
        if (some) {
          v_w1.v[e][i] = fmaf(v.v[e][i], h.v[e][i], v_w1.v[e][i]);
          if constexpr (kGate == kChannelGate) v_all.v[e][i] += z.v[e][i];
        }
        v.v[e][i] *= w1.v[e][i];
      }
    if (kGate == kRowGate && some && a.v_gate != nullptr) at.store(a.v_gate, r, a.d, z);
    if (a.w1 != nullptr) {
      float along = 0.0f, total = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          along = fmaf(v.v[e][i], h.v[e][i], along);
          total += v.v[e][i];
        }
      float2 mean = lanes.sum(along, total);
      mean.x *= at.share;
      mean.y *= at.share;
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float inner = centered ? v.v[e][i] - mean.y : v.v[e][i];
          v.v[e][i] = h_factor * fmaf(-h.v[e][i], mean.x, inner);
        }
    }
    if (some && a.v_update != nullptr) at.store(a.v_update, r, a.d, v);
  }
  float *part = a.parts + static_cast<int64_t>(blockIdx.x) * 3 * a.d;
  if (a.want_w1 != 0) store_part<T, E, kWide, kThreads, kEnd>(at, bits, a.d, v_w1, s_row, part);
  if (a.want_w2 != 0) store_part<T, E, kWide, kThreads, kEnd>(at, bits, a.d, v_w2, s_row, part + a.d);
  if constexpr (kGate == kChannelGate)
    if (a.want_gate != 0) store_part<T, E, kWide, kThreads, kEnd>(at, bits, a.d, v_all, s_row, part + 2 * a.d);
}

// The blocks' parts of up to three sums, 64 columns of one sum to a block, 16
// threads to a column.
template <typename T>
__global__ __launch_bounds__(1024) void norm_sums_kernel(const float *__restrict__ parts,
                                                         int blocks, int d, T *v_w1, T *v_w2,
                                                         T *v_gate) {
  __shared__ float s_sum[16][64];
  T *out = blockIdx.y == 0 ? v_w1 : blockIdx.y == 1 ? v_w2 : v_gate;
  if (out == nullptr) return;
  const int column = static_cast<int>(blockIdx.x) * 64 + static_cast<int>(threadIdx.x % 64);
  const int slice = static_cast<int>(threadIdx.x / 64);
  float total = 0.0f;
  if (column < d) {
    const float *p = parts + static_cast<int64_t>(blockIdx.y) * d + column;
#pragma unroll 8
    for (int b = slice; b < blocks; b += 16) total += p[static_cast<int64_t>(b) * 3 * d];
  }
  s_sum[slice][threadIdx.x % 64] = total;
  __syncthreads();
  if (slice != 0 || column >= d) return;
  for (int i = 1; i < 16; ++i) total += s_sum[i][threadIdx.x];
  out[column] = static_cast<T>(total);
}

// Lanes to a row, as a power of two, and 16-byte pieces of a lane.
struct NormForm {
  int bits, pieces;
};
NormForm norm_form(int64_t d, int type) {
  const int64_t pieces = ceil_div(d, 16 / type_size(type));
  int bits = 3, each = 1;
  while (bits < 9 && (1 << bits) < pieces) ++bits;
  while ((each << bits) < pieces) each *= 2;
  return {bits, each};
}
int norm_threads(const NormForm &f) { return f.bits > 8 ? 512 : 256; }
int64_t norm_blocks(int64_t n, const NormForm &f, int64_t most) {
  return std::max<int64_t>(1, std::min<int64_t>(most, ceil_div(n, norm_threads(f) >> f.bits)));
}
// Blocks of the backward: as many as a CU's registers hold at once, five (300k x 44
// float32: 68 us, six 83) while their parts of the sums are few bytes beside the rows,
// then three, then two.
int64_t norm_parts(int64_t n, int64_t d, const NormForm &f) {
  return norm_blocks(n, f, d <= 512 ? 1280 : d <= 1024 ? 768 : 512);
}

template <typename T, bool kBack, int E, bool kWide, int kThreads, int kGate, int kEnd>
void launch_norm_gate(const NormArgs &a, const NormForm &f, int64_t blocks, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(blocks)), block(kThreads);
  if constexpr (kBack) {
    const int groups = kThreads >> f.bits;
    const size_t lds = groups > 1 ? static_cast<size_t>(groups) * a.d * sizeof(float) : 0;
    residual_norm_bwd_kernel<T, E, kWide, kThreads, kGate, kEnd><<<grid, block, lds, stream>>>(a, f.bits);
  } else {
    residual_norm_fwd_kernel<T, E, kWide, kThreads, kGate, kEnd><<<grid, block, 0, stream>>>(a, f.bits);
  }
}
template <typename T, bool kBack, int E, bool kWide, int kThreads, int kEnd>
int launch_norm_gates(const NormArgs &a, const NormForm &f, int64_t blocks, hipStream_t stream) {
  if (a.gate_kind == kRowGate)
    launch_norm_gate<T, kBack, E, kWide, kThreads, kRowGate, kEnd>(a, f, blocks, stream);
  else if (a.gate_kind == kChannelGate)
    launch_norm_gate<T, kBack, E, kWide, kThreads, kChannelGate, kEnd>(a, f, blocks, stream);
  else
    launch_norm_gate<T, kBack, E, kWide, kThreads, kNoGate, kEnd>(a, f, blocks, stream);
  return check_launch("residual_norm");
}
template <typename T, bool kBack, int E, bool kWide, int kThreads>
int launch_norm_as(const NormArgs &a, const NormForm &f, int64_t blocks, hipStream_t stream) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  if (a.d % V == 0)
    return launch_norm_gates<T, kBack, E, kWide, kThreads, kWhole>(a, f, blocks, stream);
  if constexpr (sizeof(T) == 4) {
    return launch_norm_gates<T, kBack, E, kWide, kThreads, kElements>(a, f, blocks, stream);
  } else {
    if constexpr (!kWide)
      if (a.d < V)
        return launch_norm_gates<T, kBack, E, kWide, kThreads, kElements>(a, f, blocks, stream);
    return launch_norm_gates<T, kBack, E, kWide, kThreads, kTail>(a, f, blocks, stream);
  }
}
template <typename T, bool kBack>
int launch_norm(const NormArgs &a, const NormForm &f, int64_t blocks, hipStream_t stream) {
  if (f.bits <= 6) return launch_norm_as<T, kBack, 1, false, 256>(a, f, blocks, stream);
  if (f.bits <= 8) return launch_norm_as<T, kBack, 1, true, 256>(a, f, blocks, stream);
  if (f.pieces == 1) return launch_norm_as<T, kBack, 1, true, 512>(a, f, blocks, stream);
  if (f.pieces == 2) return launch_norm_as<T, kBack, 2, true, 512>(a, f, blocks, stream);
  if constexpr (sizeof(T) == 4) return launch_norm_as<T, kBack, 4, true, 512>(a, f, blocks, stream);
  set_error("residual_norm: no form for this width");
  return R2S_ERANGE;
}

int check_norm(const char *op, int type, int64_t n, int64_t d, const void *x, int64_t xs,
               const void *update, int64_t us, const void *gate, int64_t gs, int gate_kind,
               const void *w1) {
  R2S_REQUIRE(known_type(type), "%s: unknown element type %d", op, type);
  R2S_REQUIRE(n >= 0 && d >= 0, "%s: negative size", op);
  R2S_REQUIRE(gate_kind >= kNoGate && gate_kind <= kChannelGate, "%s: unknown gate kind %d", op,
              gate_kind);
  if (d > kNormMost || n > (int64_t{1} << 40)) {
    set_error("%s: at most %d channels and 2^40 rows", op, kNormMost);
    return R2S_ERANGE;
  }
  if (n == 0 || d == 0) return R2S_OK;
  R2S_REQUIRE(x != nullptr, "%s: null x", op);
  R2S_REQUIRE(xs >= d && (update == nullptr || us >= d) && (gate_kind != kRowGate || gs >= d),
              "%s: rows overlap", op);
  R2S_REQUIRE(gate_kind == kNoGate || gate != nullptr, "%s: null gate", op);
  R2S_REQUIRE(update != nullptr || (gate_kind == kNoGate && w1 == nullptr),
              "%s: a gate or an update's weight without an update", op);
  return R2S_OK;
}

}  // namespace
}  // namespace r2s

extern "C" {

int r2s_residual_norm_fwd(const void *x, int64_t x_stride, const void *update,
                          int64_t update_stride, const void *gate, int64_t gate_stride,
                          int32_t gate_kind, const void *update_weight, const void *weight,
                          float scale, float eps, int32_t centered, int32_t type, int64_t n,
                          int64_t width, void *y, void *u, r2s_stream_t st) {
  r2s::clear_error();
  R2S_RETURN_IF(r2s::check_norm("residual_norm_fwd", type, n, width, x, x_stride, update,
                                update_stride, gate, gate_stride, gate_kind, update_weight));
  R2S_REQUIRE(n == 0 || width == 0 || ((update != nullptr) == (y != nullptr) &&
                                       (weight != nullptr) == (u != nullptr)),
              "residual_norm_fwd: y goes with an update, u with a weight");
  if (n == 0 || width == 0 || (y == nullptr && u == nullptr)) return R2S_OK;
  r2s::NormArgs a{};
  a.x = {x, x_stride};
  a.update = {update, update_stride};
  a.gate = {gate, gate_stride};
  a.w1 = update_weight;
  a.w2 = weight;
  a.y = y;
  a.u = u;
  a.n = n;
  a.d = static_cast<int32_t>(width);
  a.gate_kind = gate_kind;
  a.centered = centered;
  a.scale = scale;
  a.eps = eps;
  const r2s::NormForm f = r2s::norm_form(width, type);
  const int64_t blocks = r2s::norm_blocks(n, f, 2048);
  R2S_BY_TYPE(type,
              return (r2s::launch_norm<T, false>(a, f, blocks, r2s::as_stream(st))));
}

int64_t r2s_residual_norm_bwd_workspace_bytes(int32_t type, int64_t n, int64_t width) {
  if (!r2s::known_type(type) || n <= 0 || width <= 0 || width > r2s::kNormMost) return 0;
  const r2s::NormForm f = r2s::norm_form(width, type);
  return r2s::norm_parts(n, width, f) * 3 * width * static_cast<int64_t>(sizeof(float));
}

int r2s_residual_norm_bwd(const void *x, int64_t x_stride, const void *update,
                          int64_t update_stride, const void *gate, int64_t gate_stride,
                          int32_t gate_kind, const void *update_weight, const void *weight,
                          const void *v_y, int64_t v_y_stride, const void *v_u,
                          int64_t v_u_stride, float scale, float eps, int32_t centered,
                          int32_t type, int64_t n, int64_t width, void *v_x, void *v_update,
                          void *v_gate, void *v_update_weight, void *v_weight, void *workspace,
                          size_t workspace_bytes, r2s_stream_t st) {
  r2s::clear_error();
  R2S_RETURN_IF(r2s::check_norm("residual_norm_bwd", type, n, width, x, x_stride, update,
                                update_stride, gate, gate_stride, gate_kind, update_weight));
  if (width == 0) return R2S_OK;
  R2S_REQUIRE((v_update == nullptr && v_update_weight == nullptr && v_gate == nullptr) ||
                  update != nullptr || n == 0,
              "residual_norm_bwd: gradients of an update that is not there");
  R2S_REQUIRE(v_update_weight == nullptr || update_weight != nullptr,
              "residual_norm_bwd: null update weight");
  R2S_REQUIRE(v_weight == nullptr || weight != nullptr, "residual_norm_bwd: null weight");
  R2S_REQUIRE(v_gate == nullptr || gate_kind != r2s::kNoGate, "residual_norm_bwd: no gate");
  R2S_REQUIRE(n == 0 || ((v_y == nullptr || v_y_stride >= width) &&
                         (v_u == nullptr || v_u_stride >= width)),
              "residual_norm_bwd: rows overlap");
  R2S_REQUIRE(v_u == nullptr || weight != nullptr, "residual_norm_bwd: v_u without a weight");
  const bool channels = gate_kind == r2s::kChannelGate;
  const bool sums = v_update_weight != nullptr || v_weight != nullptr ||
                    (channels && v_gate != nullptr);
  if (n == 0 && !sums) return R2S_OK;
  const int64_t need = r2s_residual_norm_bwd_workspace_bytes(type, n, width);
  if (sums && n > 0 && (workspace == nullptr || workspace_bytes < static_cast<size_t>(need))) {
    r2s::set_error("residual_norm_bwd: workspace of %zu bytes, %lld needed", workspace_bytes,
                   static_cast<long long>(need));
    return R2S_EWORKSPACE;
  }
  r2s::NormArgs a{};
  a.x = {x, x_stride};
  a.update = {update, update_stride};
  a.gate = {gate, gate_stride};
  a.v_y = {v_y, v_y_stride};
  a.v_u = {v_u, v_u_stride};
  a.w1 = update_weight;
  a.w2 = weight;
  a.v_x = v_x;
  a.v_update = v_update;
  a.v_gate = v_gate;
  a.parts = static_cast<float *>(workspace);
  a.n = n;
  a.d = static_cast<int32_t>(width);
  a.gate_kind = gate_kind;
  a.centered = centered;
  a.want_w1 = v_update_weight != nullptr;
  a.want_w2 = v_weight != nullptr;
  a.want_gate = channels && v_gate != nullptr;
  a.scale = scale;
  a.eps = eps;
  hipStream_t stream = r2s::as_stream(st);
  const r2s::NormForm f = r2s::norm_form(width, type);
  const int64_t blocks = n > 0 ? r2s::norm_parts(n, width, f) : 0;
  R2S_BY_TYPE(type, {
    if (n > 0) R2S_RETURN_IF((r2s::launch_norm<T, true>(a, f, blocks, stream)));
    if (!sums) return R2S_OK;
    r2s::norm_sums_kernel<T><<<dim3(static_cast<uint32_t>(r2s::ceil_div(width, 64)), 3),
                               dim3(1024), 0, stream>>>(
        a.parts, static_cast<int>(blocks), a.d, static_cast<T *>(v_update_weight),
        static_cast<T *>(v_weight), static_cast<T *>(channels ? v_gate : nullptr));
  });
  return r2s::check_launch("residual_norm_bwd sums");
}

}  // extern "C"
