// Gated linear recurrence over long sequences, and its gradient.
//
//   a_t = sigmoid(g_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t
//
// for every channel on its own, over sequences that are packed one behind
// the other; a sequence's first token has its initial state as history.
// 1 - a is computed as sigmoid(-g), so neither factor cancels.  g = +inf
// holds the state whatever x is (a term whose factor is 0 is dropped, not
// multiplied); g = -inf forgets whatever the state was.
//
// A step is the affine map h -> p h + u with p = a, u = (1 - a) x, and maps
// compose: (p2, u2) after (p1, u1) is (p2 p1, p2 u1 + u2).  A sequence's first
// token has p = 0 and its initial state inside u, which cuts the packed axis
// without any other rule.  The axis is cut into tiles; a thread composes
// kSteps steps of its channels in registers, the block composes its threads'
// maps over LDS, and the state that enters each tile comes from the tiles
// before.
//
// The gradient runs the other way.  With F_t the gradient that reaches the
// state before token t:  F_t = a_t (dy_t + F_{t+1}), again an affine map, cut
// at each sequence's last token, where F_{t+1} is the final state's gradient.
// Then with G_t = dy_t + F_{t+1}:
//   dx_t = (1 - a_t) G_t,  dg_t = a_t (1 - a_t) G_t (h_{t-1} - x_t),
// and h_{t-1} is composed again from x, g and the forward's state at the
// tile's start, which the forward keeps (one state per tile, float32).
//
// The reverse order is the same code on mirrored token and sequence numbers.
#include "r2s_latent.h"

namespace r2s {
namespace {

constexpr int kThreads = 256;
constexpr int kSteps = 16;  // tokens per thread

// What every kernel of a call needs to know of its tokens.  Tokens and
// sequences are numbered in scan order; physical numbers are mirrored with
// `reverse`.  offsets null: sequences of `length` tokens.
struct Tokens {
  const int32_t *offsets;
  int64_t n, length;
  int32_t sequences;
  int32_t reverse;
  uint32_t width;
  uint32_t lane_bits;  // 2^lane_bits lanes across a tile's channels
  int32_t tiles;

  __device__ __forceinline__ int64_t start(int64_t s) const {
    if (offsets == nullptr) return s * length;
    return reverse ? n - offsets[sequences - s] : offsets[s];
  }
  __device__ __forceinline__ int64_t row(int64_t t) const { return reverse ? n - 1 - t : t; }
  __device__ __forceinline__ int64_t state_row(int64_t s) const {
    return reverse ? sequences - 1 - s : s;
  }
  __device__ __forceinline__ int groups() const { return kThreads >> lane_bits; }
  __device__ __forceinline__ int tile_tokens() const { return groups() * kSteps; }
};

// sigmoid(g) and sigmoid(-g), each to a few units in its own last place.
__device__ __forceinline__ void gate_pair(float g, float &a, float &b) {
  const float e = __builtin_amdgcn_exp2f(fabsf(g) * -1.44269504088896341f);
  const float r = __builtin_amdgcn_rcpf(1.0f + e), q = e * r;
  a = g < 0.0f ? q : r;
  b = g < 0.0f ? r : q;
}

// factor * value, with a factor of 0 taking any value (also a NaN) to 0.
__device__ __forceinline__ float scaled(float factor, float value) {
  return factor == 0.0f ? 0.0f : factor * value;
}
// p h + u, likewise.
__device__ __forceinline__ float applied(float p, float h, float u) {
  return p == 0.0f ? u : fmaf(p, h, u);
}

// s_first[t]: the sequence whose first token is the tile's token t, else -1
// (also for the places of a last tile that no token has); s_last likewise.
__device__ __forceinline__ void mark_sequences(const Tokens &c, int64_t t0, int32_t *s_first,
                                               int32_t *s_last) {
  __shared__ int32_t s_seq;
  const int places = c.tile_tokens();
  const int count = static_cast<int>(min(static_cast<int64_t>(places), c.n - t0));
  for (int t = threadIdx.x; t < places; t += kThreads) s_first[t] = s_last[t] = -1;
  if (c.offsets == nullptr) {
    __syncthreads();
    for (int t = threadIdx.x; t < count; t += kThreads) {
      const int64_t s = (t0 + t) / c.length, in = t0 + t - s * c.length;
      if (in == 0) s_first[t] = static_cast<int32_t>(s);
      if (in == c.length - 1) s_last[t] = static_cast<int32_t>(s);
    }
    __syncthreads();
    return;
  }
  if (threadIdx.x < 64) {
    // The last sequence that starts at or before t0: 64 probes a round.
    int64_t lo = 0, hi = c.sequences;  // start(lo) <= t0 (or lo = 0), start(hi) > t0 (or the end)
    while (hi - lo > 1) {
      const int64_t step = (hi - lo + 63) / 64;
      const int64_t s = lo + (static_cast<int64_t>(threadIdx.x) + 1) * step;
      const uint64_t under = ballot(s < hi && c.start(s) <= t0);
      const int64_t k = __popcll(under);
      hi = min(hi, lo + (k + 1) * step);
      lo += k * step;
    }
    if (threadIdx.x == 0) s_seq = static_cast<int32_t>(lo);
  }
  __syncthreads();
  // Every sequence with a token in the tile, 256 at a time, to the first that
  // starts past it.
  const int64_t end = t0 + count;
  for (int64_t s = s_seq;; s += kThreads) {
    const int64_t mine = s + threadIdx.x;
    int64_t lo = end;
    if (mine < c.sequences) {
      lo = c.start(mine);
      const int64_t hi = c.start(mine + 1);
      if (lo < hi) {
        if (lo >= t0 && lo < end) s_first[lo - t0] = static_cast<int32_t>(mine);
        if (hi - 1 >= t0 && hi - 1 < end) s_last[hi - 1 - t0] = static_cast<int32_t>(mine);
      }
    }
    if (!__syncthreads_or(threadIdx.x == kThreads - 1 && lo < end &&
                          s + kThreads < c.sequences))
      break;
  }
}

// A thread's place in its tile.
struct Place {
  int group;       // of kSteps tokens
  uint32_t col;    // its first channel
  uint32_t lane;   // among the lanes across the channels
  bool inside;     // the channels exist
  __device__ __forceinline__ Place(const Tokens &c, int V) {
    lane = threadIdx.x & ((1u << c.lane_bits) - 1u);
    group = static_cast<int>(threadIdx.x >> c.lane_bits);
    col = ((blockIdx.y << c.lane_bits) + lane) * V;
    inside = col < c.width;
  }
};

template <typename T, int V>
__device__ __forceinline__ void load_rows(const T *p, int64_t stride, const Tokens &c,
                                          const Place &at, int64_t t0, Pack<T, V> (&x)[kSteps]) {
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int64_t t = t0 + at.group * kSteps + k;
    if (at.inside && t < c.n) {
      x[k] = load_pack<T, V>(p + c.row(t) * stride + at.col);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) x[k].v[v] = static_cast<T>(0.0f);
    }
  }
}

// One forward step's map.  first: the sequence that begins here, or -1.
__device__ __forceinline__ void forward_step(float x, float g, float h0, bool first, float &p,
                                             float &u) {
  float b;
  gate_pair(g, p, b);
  u = scaled(b, x);
  if (first) {
    u = applied(p, h0, u);
    p = 0.0f;
  }
}

// ------------------------------------------------------------- forward ---

// The map of each tile: maps [tiles][2][width].
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void scan_fwd_maps_kernel(
    const T *__restrict__ x, int64_t x_stride, const T *__restrict__ gate, int64_t g_stride,
    const float *__restrict__ initial, Tokens c, float *__restrict__ maps) {
  __shared__ int32_t s_first[kThreads * kSteps], s_last[kThreads * kSteps];
  __shared__ float s_p[kThreads * V], s_u[kThreads * V];
  const Place at(c, V);
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * c.tile_tokens();
  mark_sequences(c, t0, s_first, s_last);
  Pack<T, V> xs[kSteps], gs[kSteps];
  load_rows<T, V>(x, x_stride, c, at, t0, xs);
  load_rows<T, V>(gate, g_stride, c, at, t0, gs);
  float p[V], u[V];
#pragma unroll
  for (int v = 0; v < V; ++v) p[v] = 1.0f, u[v] = 0.0f;
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    if (t0 + at.group * kSteps + k < c.n) {
      const int32_t s = s_first[at.group * kSteps + k];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float h0 = 0.0f, pk, uk;
        if (s >= 0 && initial != nullptr && at.inside)
          h0 = initial[c.state_row(s) * c.width + at.col + v];
        forward_step(static_cast<float>(xs[k].v[v]), static_cast<float>(gs[k].v[v]), h0, s >= 0,
                     pk, uk);
        u[v] = applied(pk, u[v], uk);
        p[v] = p[v] * pk;
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) s_p[threadIdx.x * V + v] = p[v], s_u[threadIdx.x * V + v] = u[v];
  __syncthreads();
  if (at.group != 0 || !at.inside) return;
  for (int q = 1; q < c.groups(); ++q) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = ((q << c.lane_bits) + static_cast<int>(at.lane)) * V + v;
      u[v] = applied(s_p[i], u[v], s_u[i]);
      p[v] *= s_p[i];
    }
  }
  float *m = maps + static_cast<int64_t>(blockIdx.x) * 2 * c.width + at.col;
#pragma unroll
  for (int v = 0; v < V; ++v) m[v] = p[v], m[c.width + v] = u[v];
}

// The state that enters each tile, from the tiles' maps in order (from the
// last tile down with `down`).  A block takes 16 channels; each of its 16
// rows of threads composes one sixteenth of the tiles, and again with the
// state that the rows before leave.
__global__ __launch_bounds__(kThreads) void scan_carry_kernel(const float *__restrict__ maps,
                                                              int32_t tiles, uint32_t width,
                                                              int32_t down,
                                                              float *__restrict__ carries) {
  __shared__ float s_p[16][16], s_u[16][16];
  const uint32_t lane = threadIdx.x % 16, row = threadIdx.x / 16;
  const uint32_t col = blockIdx.x * 16 + lane;
  const int32_t per = (tiles + 15) / 16, i0 = static_cast<int32_t>(row) * per;
  const int32_t i1 = min(i0 + per, tiles);
  const bool inside = col < width;
  auto at = [&](int32_t i) { return static_cast<int64_t>(down ? tiles - 1 - i : i); };
  float p = 1.0f, u = 0.0f;
  if (inside) {
#pragma unroll 8
    for (int32_t i = i0; i < i1; ++i) {
      const float *m = maps + at(i) * 2 * width + col;
      u = applied(m[0], u, m[width]);
      p *= m[0];
    }
  }
  s_p[row][lane] = p;
  s_u[row][lane] = u;
  __syncthreads();
  if (!inside) return;
  float h = 0.0f;
  for (uint32_t r = 0; r < row; ++r) h = applied(s_p[r][lane], h, s_u[r][lane]);
#pragma unroll 8
  for (int32_t i = i0; i < i1; ++i) {
    const float *m = maps + at(i) * 2 * width + col;
    carries[at(i) * width + col] = h;
    h = applied(m[0], h, m[width]);
  }
}

// The threads' own incoming values from the block's: composes the maps that
// the threads left in s_p, s_u, in group order (downwards with kDown).
template <int V, bool kDown>
__device__ __forceinline__ void enter(const Tokens &c, const Place &at, const float *s_p,
                                      const float *s_u, float (&h)[V]) {
  const int count = kDown ? c.groups() - 1 - at.group : at.group;
  for (int i = 0; i < count; ++i) {
    const int q = kDown ? c.groups() - 1 - i : i;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int j = ((q << c.lane_bits) + static_cast<int>(at.lane)) * V + v;
      h[v] = applied(s_p[j], h[v], s_u[j]);
    }
  }
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void scan_fwd_apply_kernel(
    const T *__restrict__ x, int64_t x_stride, const T *__restrict__ gate, int64_t g_stride,
    const float *__restrict__ initial, Tokens c, const float *__restrict__ carries,
    T *__restrict__ y, float *__restrict__ final) {
  __shared__ int32_t s_first[kThreads * kSteps], s_last[kThreads * kSteps];
  __shared__ float s_p[kThreads * V], s_u[kThreads * V];
  const Place at(c, V);
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * c.tile_tokens();
  mark_sequences(c, t0, s_first, s_last);
  Pack<T, V> xs[kSteps], gs[kSteps];
  load_rows<T, V>(x, x_stride, c, at, t0, xs);
  load_rows<T, V>(gate, g_stride, c, at, t0, gs);
  // Each step's map composed with the thread's steps before it.
  float p[kSteps][V], u[kSteps][V];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int32_t s = s_first[at.group * kSteps + k];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float h0 = 0.0f;
      if (s >= 0 && initial != nullptr && at.inside)
        h0 = initial[c.state_row(s) * c.width + at.col + v];
      forward_step(static_cast<float>(xs[k].v[v]), static_cast<float>(gs[k].v[v]), h0, s >= 0,
                   p[k][v], u[k][v]);
      if (k > 0) {
        u[k][v] = applied(p[k][v], u[k - 1][v], u[k][v]);
        p[k][v] *= p[k - 1][v];
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s_p[threadIdx.x * V + v] = p[kSteps - 1][v];
    s_u[threadIdx.x * V + v] = u[kSteps - 1][v];
  }
  __syncthreads();
  if (!at.inside) return;
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v)
    h[v] = carries[static_cast<int64_t>(blockIdx.x) * c.width + at.col + v];
  enter<V, false>(c, at, s_p, s_u, h);
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int64_t t = t0 + at.group * kSteps + k;
    if (t >= c.n) break;
    Pack<T, V> out;
    const int32_t s = s_last[at.group * kSteps + k];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float state = applied(p[k][v], h[v], u[k][v]);
      out.v[v] = static_cast<T>(state);
      if (s >= 0) final[c.state_row(s) * c.width + at.col + v] = state;
    }
    store_pack<T, V>(y + c.row(t) * c.width + at.col, out);
  }
}

// Sequences without a token: the state they end in (or its gradient) is the
// one they began with.
__global__ __launch_bounds__(kThreads) void scan_empty_kernel(Tokens c,
                                                              const float *__restrict__ in,
                                                              float *__restrict__ out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t s = i / c.width;
  if (s >= c.sequences || (c.offsets != nullptr && c.offsets[s] < c.offsets[s + 1])) return;
  out[i] = in != nullptr ? in[i] : 0.0f;
}

// One token per sequence, the decode form: nothing to scan.
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void scan_step_kernel(
    const T *__restrict__ x, int64_t x_stride, const T *__restrict__ gate, int64_t g_stride,
    const float *__restrict__ initial, int64_t n, uint32_t width, T *__restrict__ y,
    float *__restrict__ final) {
  const uint32_t vpr = width / V;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t t = i / vpr;
  if (t >= n) return;
  const uint32_t col = static_cast<uint32_t>(i - t * vpr) * V;
  const Pack<T, V> xs = load_pack<T, V>(x + t * x_stride + col);
  const Pack<T, V> gs = load_pack<T, V>(gate + t * g_stride + col);
  Pack<T, V> out;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float h0 = initial != nullptr ? initial[t * width + col + v] : 0.0f;
    float p, u;
    forward_step(static_cast<float>(xs.v[v]), static_cast<float>(gs.v[v]), h0, true, p, u);
    out.v[v] = static_cast<T>(u);
    final[t * width + col + v] = u;
  }
  store_pack<T, V>(y + t * width + col, out);
}

// ------------------------------------------------------------ backward ---

// F_t = a_t (dy_t + F_{t+1}) as a map of F_{t+1}; the last token of a
// sequence takes the final state's gradient and no other.
__device__ __forceinline__ void backward_step(float a, float dy, float last_grad, bool last,
                                              float &p, float &u) {
  p = last ? 0.0f : a;
  u = scaled(a, last ? dy + last_grad : dy);
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void scan_bwd_maps_kernel(
    const T *__restrict__ gate, int64_t g_stride, const T *__restrict__ v_y, int64_t v_stride,
    const float *__restrict__ v_final, Tokens c, float *__restrict__ maps) {
  __shared__ int32_t s_first[kThreads * kSteps], s_last[kThreads * kSteps];
  __shared__ float s_p[kThreads * V], s_u[kThreads * V];
  const Place at(c, V);
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * c.tile_tokens();
  mark_sequences(c, t0, s_first, s_last);
  Pack<T, V> gs[kSteps], vs[kSteps];
  load_rows<T, V>(gate, g_stride, c, at, t0, gs);
  load_rows<T, V>(v_y, v_stride, c, at, t0, vs);
  float p[V], u[V];
#pragma unroll
  for (int v = 0; v < V; ++v) p[v] = 1.0f, u[v] = 0.0f;
#pragma unroll
  for (int k = kSteps - 1; k >= 0; --k) {
    if (t0 + at.group * kSteps + k < c.n) {
      const int32_t s = s_last[at.group * kSteps + k];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float vf = 0.0f, a, b, pk, uk;
        if (s >= 0 && v_final != nullptr && at.inside)
          vf = v_final[c.state_row(s) * c.width + at.col + v];
        gate_pair(static_cast<float>(gs[k].v[v]), a, b);
        backward_step(a, static_cast<float>(vs[k].v[v]), vf, s >= 0, pk, uk);
        u[v] = applied(pk, u[v], uk);
        p[v] *= pk;
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) s_p[threadIdx.x * V + v] = p[v], s_u[threadIdx.x * V + v] = u[v];
  __syncthreads();
  if (at.group != c.groups() - 1 || !at.inside) return;
  for (int q = c.groups() - 2; q >= 0; --q) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = ((q << c.lane_bits) + static_cast<int>(at.lane)) * V + v;
      u[v] = applied(s_p[i], u[v], s_u[i]);
      p[v] *= s_p[i];
    }
  }
  float *m = maps + static_cast<int64_t>(blockIdx.x) * 2 * c.width + at.col;
#pragma unroll
  for (int v = 0; v < V; ++v) m[v] = p[v], m[c.width + v] = u[v];
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void scan_bwd_apply_kernel(
    const T *__restrict__ x, int64_t x_stride, const T *__restrict__ gate, int64_t g_stride,
    const float *__restrict__ initial, const T *__restrict__ v_y, int64_t v_stride,
    const float *__restrict__ v_final, Tokens c, const float *__restrict__ carries,
    const float *__restrict__ flows, T *__restrict__ v_x, T *__restrict__ v_gate,
    float *__restrict__ v_initial) {
  __shared__ int32_t s_first[kThreads * kSteps], s_last[kThreads * kSteps];
  __shared__ float s_p[kThreads * V], s_u[kThreads * V];
  const Place at(c, V);
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * c.tile_tokens();
  mark_sequences(c, t0, s_first, s_last);
  Pack<T, V> xs[kSteps], gs[kSteps], vs[kSteps];
  load_rows<T, V>(x, x_stride, c, at, t0, xs);
  load_rows<T, V>(gate, g_stride, c, at, t0, gs);
  load_rows<T, V>(v_y, v_stride, c, at, t0, vs);
  const int32_t *first = s_first + at.group * kSteps, *last = s_last + at.group * kSteps;
  auto state0 = [&](int k, int v) {
    return first[k] >= 0 && initial != nullptr && at.inside
               ? initial[c.state_row(first[k]) * c.width + at.col + v]
               : 0.0f;
  };
  auto grad0 = [&](int k, int v) {
    return last[k] >= 0 && v_final != nullptr && at.inside
               ? v_final[c.state_row(last[k]) * c.width + at.col + v]
               : 0.0f;
  };
  // Both scans' maps over the thread's tokens.
  float hp[V], hu[V], fp[V], fu[V];
#pragma unroll
  for (int v = 0; v < V; ++v) hp[v] = fp[v] = 1.0f, hu[v] = fu[v] = 0.0f;
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float p, u;
      forward_step(static_cast<float>(xs[k].v[v]), static_cast<float>(gs[k].v[v]), state0(k, v),
                   first[k] >= 0, p, u);
      hu[v] = applied(p, hu[v], u);
      hp[v] *= p;
    }
  }
#pragma unroll
  for (int k = kSteps - 1; k >= 0; --k) {
    if (t0 + at.group * kSteps + k < c.n) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a, b, p, u;
        gate_pair(static_cast<float>(gs[k].v[v]), a, b);
        backward_step(a, static_cast<float>(vs[k].v[v]), grad0(k, v), last[k] >= 0, p, u);
        fu[v] = applied(p, fu[v], u);
        fp[v] *= p;
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) s_p[threadIdx.x * V + v] = hp[v], s_u[threadIdx.x * V + v] = hu[v];
  __syncthreads();
  float h[V], f[V];
  const int64_t tile = static_cast<int64_t>(blockIdx.x) * c.width + at.col;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    h[v] = at.inside ? carries[tile + v] : 0.0f;
    f[v] = at.inside ? flows[tile + v] : 0.0f;
  }
  enter<V, false>(c, at, s_p, s_u, h);
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) s_p[threadIdx.x * V + v] = fp[v], s_u[threadIdx.x * V + v] = fu[v];
  __syncthreads();
  enter<V, true>(c, at, s_p, s_u, f);
  if (!at.inside) return;
  // The states before each token, then the tokens from the last to the first.
  float prior[kSteps][V];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a, b;
      gate_pair(static_cast<float>(gs[k].v[v]), a, b);
      prior[k][v] = first[k] >= 0 ? state0(k, v) : h[v];
      h[v] = applied(a, prior[k][v], scaled(b, static_cast<float>(xs[k].v[v])));
    }
  }
#pragma unroll
  for (int k = kSteps - 1; k >= 0; --k) {
    const int64_t t = t0 + at.group * kSteps + k;
    if (t < c.n) {
      Pack<T, V> vx, vg;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a, b;
        gate_pair(static_cast<float>(gs[k].v[v]), a, b);
        const float g = static_cast<float>(vs[k].v[v]) + (last[k] >= 0 ? grad0(k, v) : f[v]);
        vx.v[v] = static_cast<T>(scaled(b, g));
        vg.v[v] = static_cast<T>(
            scaled(a * b, g * (prior[k][v] - static_cast<float>(xs[k].v[v]))));
        f[v] = scaled(a, g);
        if (first[k] >= 0 && v_initial != nullptr)
          v_initial[c.state_row(first[k]) * c.width + at.col + v] = f[v];
      }
      store_pack<T, V>(v_x + c.row(t) * c.width + at.col, vx);
      store_pack<T, V>(v_gate + c.row(t) * c.width + at.col, vg);
    }
  }
}

// ---------------------------------------------------------------- host ---

// Lanes across the channels, for vectors of V.
uint32_t lane_bits_for(int64_t width, int V) {
  const int64_t vpr = ceil_div(width, V);
  uint32_t bits = 0;
  while (bits < 6 && (1 << bits) < vpr) ++bits;
  return bits;
}

int vector_for(int type, int64_t width) {
  // 4 bytes of 16-bit elements where the width is even; see the strides' check
  // of the caller.
  return type == R2S_TYPE_F32 ? 1 : (width % 2 == 0 ? 2 : 1);
}

int64_t tile_count(int type, int64_t n, int64_t width) {
  const int V = vector_for(type, width);
  return ceil_div(n, static_cast<int64_t>(kThreads >> lane_bits_for(width, V)) * kSteps);
}

struct ScanSpace {
  float *maps, *flows;
};
ScanSpace carve_scan(Carver &cv, int64_t tiles, int64_t width, bool backward) {
  ScanSpace s;
  s.maps = cv.take<float>(tiles * 2 * width);
  s.flows = backward ? cv.take<float>(tiles * width) : nullptr;
  return s;
}

int check_scan(const char *what, int type, const int32_t *offsets, int64_t n, int64_t sequences,
               int64_t length, int64_t width) {
  R2S_REQUIRE(known_type(type), "%s: unknown element type %d", what, type);
  R2S_REQUIRE(n >= 0 && sequences >= 0 && length >= 0 && width >= 0, "%s: negative size", what);
  R2S_REQUIRE(offsets != nullptr || n == sequences * length,
              "%s: %lld tokens are not %lld sequences of %lld", what, (long long)n,
              (long long)sequences, (long long)length);
  R2S_REQUIRE(sequences > 0 || n == 0, "%s: tokens without a sequence", what);
  if (n > kInt32Max || sequences >= kInt32Max || width > (1 << 20)) {
    set_error("%s: more than 2^31 - 1 tokens or sequences, or more than 2^20 channels", what);
    return R2S_ERANGE;
  }
  return R2S_OK;
}

Tokens tokens_of(int type, const int32_t *offsets, int64_t n, int64_t sequences, int64_t length,
                 int64_t width, int32_t reverse) {
  Tokens c{};
  c.offsets = offsets;
  c.n = n;
  c.length = length;
  c.sequences = static_cast<int32_t>(sequences);
  c.reverse = reverse != 0;
  c.width = static_cast<uint32_t>(width);
  c.lane_bits = lane_bits_for(width, vector_for(type, width));
  c.tiles = static_cast<int32_t>(tile_count(type, n, width));
  return c;
}

dim3 scan_grid(const Tokens &c, int V) {
  return dim3(static_cast<uint32_t>(c.tiles),
              static_cast<uint32_t>(ceil_div(c.width, static_cast<int64_t>(V) << c.lane_bits)));
}

int empty_states(const Tokens &c, const float *in, float *out, hipStream_t stream) {
  const int64_t blocks = ceil_div(static_cast<int64_t>(c.sequences) * c.width, kThreads);
  if (blocks == 0 || (c.offsets == nullptr && c.length > 0)) return R2S_OK;
  scan_empty_kernel<<<dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, stream>>>(c, in,
                                                                                         out);
  return check_launch("gated_scan empty sequences");
}

int carry(const Tokens &c, const float *maps, bool down, float *out, hipStream_t stream) {
  scan_carry_kernel<<<dim3(static_cast<uint32_t>(ceil_div(c.width, 16))), dim3(kThreads), 0,
                      stream>>>(maps, c.tiles, c.width, down, out);
  return check_launch("gated_scan carries");
}

template <typename T, int V>
int scan_fwd(const Tokens &c, const void *x, int64_t xs, const void *g, int64_t gs,
             const float *initial, void *y, float *final, float *carries, const ScanSpace &s,
             hipStream_t stream) {
  const T *xt = static_cast<const T *>(x), *gt = static_cast<const T *>(g);
  if (c.offsets == nullptr && c.length == 1) {
    const int64_t blocks = ceil_div(c.n * (c.width / V), kThreads);
    if (blocks > kInt32Max) {
      set_error("gated_scan_fwd: too many tokens");
      return R2S_ERANGE;
    }
    scan_step_kernel<T, V><<<dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, stream>>>(
        xt, xs, gt, gs, initial, c.n, c.width, static_cast<T *>(y), final);
    return check_launch("gated_scan_fwd");
  }
  const dim3 grid = scan_grid(c, V);
  scan_fwd_maps_kernel<T, V><<<grid, dim3(kThreads), 0, stream>>>(xt, xs, gt, gs, initial, c,
                                                                  s.maps);
  R2S_RETURN_IF(check_launch("gated_scan_fwd"));
  R2S_RETURN_IF(carry(c, s.maps, false, carries, stream));
  scan_fwd_apply_kernel<T, V><<<grid, dim3(kThreads), 0, stream>>>(
      xt, xs, gt, gs, initial, c, carries, static_cast<T *>(y), final);
  return check_launch("gated_scan_fwd");
}

template <typename T, int V>
int scan_bwd(const Tokens &c, const void *x, int64_t xs, const void *g, int64_t gs,
             const float *initial, const float *carries, const void *v_y, int64_t vs,
             const float *v_final, void *v_x, void *v_gate, float *v_initial, const ScanSpace &s,
             hipStream_t stream) {
  const T *xt = static_cast<const T *>(x), *gt = static_cast<const T *>(g);
  const T *vt = static_cast<const T *>(v_y);
  const dim3 grid = scan_grid(c, V);
  scan_bwd_maps_kernel<T, V><<<grid, dim3(kThreads), 0, stream>>>(gt, gs, vt, vs, v_final, c,
                                                                  s.maps);
  R2S_RETURN_IF(check_launch("gated_scan_bwd"));
  R2S_RETURN_IF(carry(c, s.maps, true, s.flows, stream));
  scan_bwd_apply_kernel<T, V><<<grid, dim3(kThreads), 0, stream>>>(
      xt, xs, gt, gs, initial, vt, vs, v_final, c, carries, s.flows, static_cast<T *>(v_x),
      static_cast<T *>(v_gate), v_initial);
  return check_launch("gated_scan_bwd");
}

// Whether rows may be read two 16-bit elements at a time.
bool pairs_fit(std::initializer_list<const void *> bases, std::initializer_list<int64_t> strides) {
  for (const void *p : bases)
    if (address(p) % 4 != 0) return false;
  for (int64_t s : strides)
    if (s % 2 != 0) return false;
  return true;
}

}  // namespace
}  // namespace r2s

extern "C" {

int64_t r2s_gated_scan_tiles(int32_t type, int64_t n, int64_t width) {
  if (!r2s::known_type(type) || n <= 0 || width <= 0) return 0;
  return r2s::tile_count(type, n, width);
}

int64_t r2s_gated_scan_workspace_bytes(int32_t type, int64_t n, int64_t width, int32_t backward) {
  r2s::Carver cv(nullptr);
  r2s::carve_scan(cv, r2s_gated_scan_tiles(type, n, width), width > 0 ? width : 0, backward != 0);
  return static_cast<int64_t>(cv.used);
}

int r2s_gated_scan_fwd(const void *x, int64_t x_stride, const void *gate, int64_t gate_stride,
                       const float *initial, const int32_t *offsets, int64_t sequences,
                       int64_t length, int64_t n, int64_t width, int32_t type, int32_t reverse,
                       void *y, float *final_state, float *carries, void *ws, size_t ws_bytes,
                       r2s_stream_t st) {
  using namespace r2s;
  clear_error();
  R2S_RETURN_IF(check_scan("gated_scan_fwd", type, offsets, n, sequences, length, width));
  if (width == 0 || sequences == 0) return R2S_OK;
  R2S_REQUIRE(x_stride >= width && gate_stride >= width, "gated_scan_fwd: rows overlap");
  R2S_REQUIRE(final_state != nullptr, "gated_scan_fwd: null final states");
  const Tokens c = tokens_of(type, offsets, n, sequences, length, width, reverse);
  hipStream_t stream = as_stream(st);
  R2S_RETURN_IF(empty_states(c, initial, final_state, stream));
  if (n == 0) return R2S_OK;
  R2S_REQUIRE(x != nullptr && gate != nullptr && y != nullptr && carries != nullptr,
              "gated_scan_fwd: null tokens, outputs or carries");
  const int64_t need = r2s_gated_scan_workspace_bytes(type, n, width, 0);
  if (ws == nullptr || static_cast<int64_t>(ws_bytes) < need) {
    set_error("gated_scan_fwd: workspace of %zu bytes, %lld required", ws_bytes, (long long)need);
    return R2S_EWORKSPACE;
  }
  Carver cv(ws);
  const ScanSpace s = carve_scan(cv, c.tiles, width, false);
  const int V = vector_for(type, width);
  R2S_REQUIRE(V == 1 || pairs_fit({x, gate, y}, {x_stride, gate_stride}),
              "gated_scan_fwd: rows of 16-bit elements must start at multiples of 4 bytes");
  R2S_BY_TYPE(type, {
    if constexpr (sizeof(T) == 2) {
      if (V == 2)
        return scan_fwd<T, 2>(c, x, x_stride, gate, gate_stride, initial, y, final_state, carries,
                              s, stream);
    }
    return scan_fwd<T, 1>(c, x, x_stride, gate, gate_stride, initial, y, final_state, carries, s,
                          stream);
  });
  return R2S_OK;
}

int r2s_gated_scan_bwd(const void *x, int64_t x_stride, const void *gate, int64_t gate_stride,
                       const float *initial, const int32_t *offsets, const float *carries,
                       const void *v_y, int64_t v_y_stride, const float *v_final,
                       int64_t sequences, int64_t length, int64_t n, int64_t width, int32_t type,
                       int32_t reverse, void *v_x, void *v_gate, float *v_initial, void *ws,
                       size_t ws_bytes, r2s_stream_t st) {
  using namespace r2s;
  clear_error();
  R2S_RETURN_IF(check_scan("gated_scan_bwd", type, offsets, n, sequences, length, width));
  if (width == 0 || sequences == 0) return R2S_OK;
  R2S_REQUIRE(x_stride >= width && gate_stride >= width && v_y_stride >= width,
              "gated_scan_bwd: rows overlap");
  const Tokens c = tokens_of(type, offsets, n, sequences, length, width, reverse);
  hipStream_t stream = as_stream(st);
  if (v_initial != nullptr) R2S_RETURN_IF(empty_states(c, v_final, v_initial, stream));
  if (n == 0) return R2S_OK;
  R2S_REQUIRE(x != nullptr && gate != nullptr && v_y != nullptr && carries != nullptr &&
                  v_x != nullptr && v_gate != nullptr,
              "gated_scan_bwd: null tokens, gradients or carries");
  const int64_t need = r2s_gated_scan_workspace_bytes(type, n, width, 1);
  if (ws == nullptr || static_cast<int64_t>(ws_bytes) < need) {
    set_error("gated_scan_bwd: workspace of %zu bytes, %lld required", ws_bytes, (long long)need);
    return R2S_EWORKSPACE;
  }
  Carver cv(ws);
  const ScanSpace s = carve_scan(cv, c.tiles, width, true);
  const int V = vector_for(type, width);
  R2S_REQUIRE(V == 1 || pairs_fit({x, gate, v_y, v_x, v_gate},
                                  {x_stride, gate_stride, v_y_stride}),
              "gated_scan_bwd: rows of 16-bit elements must start at multiples of 4 bytes");
  R2S_BY_TYPE(type, {
    if constexpr (sizeof(T) == 2) {
      if (V == 2)
        return scan_bwd<T, 2>(c, x, x_stride, gate, gate_stride, initial, carries, v_y, v_y_stride,
                              v_final, v_x, v_gate, v_initial, s, stream);
    }
    return scan_bwd<T, 1>(c, x, x_stride, gate, gate_stride, initial, carries, v_y, v_y_stride,
                          v_final, v_x, v_gate, v_initial, s, stream);
  });
  return R2S_OK;
}

}  // extern "C"
