// Gated linear recurrence over long sequences, and its gradient.
//
//   a_t = sigmoid(g_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t
//
// for every channel on its own, over sequences that are packed one behind
// the other; a sequence's first token has its initial state as history.
// 1 - a is computed as sigmoid(-g), so neither factor cancels.  g = +inf
// holds the state whatever x is (a term whose factor is 0 is dropped, not
// multiplied); g = -inf forgets whatever the state was.  So do finite gates
// beyond 87.3, whose smaller factor is below float32's normal range: it is 0.
//
// A step is the affine map h -> p h + u with p = a, u = (1 - a) x, and maps
// compose: (p2, u2) after (p1, u1) is (p2 p1, p2 u1 + u2).  A sequence's first
// token has p = 0 and its initial state inside u, which cuts the packed axis
// without any other rule.  p is never negative, so its sign bit marks a map
// that has such a cut in it, or a gate that forgets: nothing of the state before
// it goes through, not a NaN either.  A product of gates that merely falls below
// float32's range stays at its smallest number, 2^-149, and lets through what is
// not finite.  So the axis is cut into strips of equal length
// whatever the sequences are.  A group of lanes (one vector of channels each)
// walks one strip, token after token, in registers: once to compose the
// strip's map, then, with the state that enters the strip, to write the
// states.  No step of either walk waits for another lane.
//
//   rounds     a block holds whole sequences (one of equal ones, or all of a
//              few) and walks them 8 tokens per group at a time: tokens are
//              read once, everything is one launch.
//   packed     a launch composes the strips' maps, one adds them up along the
//              axis, one walks again: for few long sequences and ragged ones,
//              whose lengths only the device knows.
//   own        short equal sequences: a strip is a sequence, one walk.
//
// The gradient runs the other way.  With F_t the gradient that reaches the
// state before token t:  F_t = a_t (dy_t + F_{t+1}), again an affine map, cut
// at each sequence's last token, where F_{t+1} is the final state's gradient.
// Then with G_t = dy_t + F_{t+1}:
//   dx_t = (1 - a_t) G_t,  dg_t = a_t (1 - a_t) G_t (h_{t-1} - x_t),
// and h_{t-1} is composed again from x, g and the state before each kChunk
// tokens, which the forward keeps in float32.
//
// The reverse order is the same code on mirrored token and sequence numbers.
// The plain and the careful form of each walk round alike (no contraction but
// the fmaf written), so a token's bits do not depend on its neighbours'.
#pragma clang fp contract(off)

#include <algorithm>

#include "r2s_latent.h"

namespace r2s {
namespace {

constexpr int kThreads = 256;  // of a block of strips
constexpr int kRoundThreads = 512;  // of a block that walks in rounds, at most
constexpr int kChunk = 8;        // tokens loaded together, and between kept states

// What every kernel of a call needs to know of its tokens.  Tokens and
// sequences are numbered in scan order; physical numbers are mirrored with
// `reverse`.  offsets null: sequences of `length` tokens.
// Strip i of block b holds tokens [b block + i strip, + strip), not past the
// block's.
struct Tokens {
  const int32_t *offsets;
  int64_t n, length;
  int64_t block;       // tokens per block
  int32_t sequences;
  int32_t reverse;
  int32_t strip;       // tokens per strip
  int32_t steps;       // the same, to the next multiple of kChunk
  uint32_t width;
  uint32_t lane_bits;  // 2^lane_bits lanes across a block's channels

  __device__ __forceinline__ int64_t start(int64_t s) const {
    if (offsets == nullptr) return s * length;
    return reverse ? n - offsets[sequences - s] : offsets[s];
  }
  __device__ __forceinline__ int64_t state_row(int64_t s) const {
    return reverse ? sequences - 1 - s : s;
  }
};

// sigmoid(g) and sigmoid(-g).  The exponent is rounded before exp2, so the smaller
// one is good to 2 |g| + 6 units of 2^-24 (|g| below 87.3; 0 beyond, where exp2
// returns no subnormal numbers), the larger to a few.
__device__ __forceinline__ void gate_pair(float g, float &a, float &b) {
  const float e = __builtin_amdgcn_exp2f(fabsf(g) * -1.44269504088896341f);
  const float r = __builtin_amdgcn_rcpf(1.0f + e), q = e * r;
  a = g < 0.0f ? q : r;
  b = g < 0.0f ? r : q;
}

// factor * value, with a factor of 0 taking any value (also a NaN) to 0; only
// with kSafe, where a chunk holds something that is not finite.
template <bool kSafe>
__device__ __forceinline__ float scaled(float factor, float value) {
  return kSafe && factor == 0.0f ? 0.0f : factor * value;
}
// a h + u for a token's factor a, likewise.
template <bool kSafe>
__device__ __forceinline__ float applied(float a, float h, float u) {
  return kSafe && a == 0.0f ? u : fmaf(a, h, u);
}

__device__ __forceinline__ bool finite(float x) { return __builtin_isfinite(x); }

// A map's factor p, with its sign bit as the mark of a cut: a product that may
// have left the range, two maps together, and the state behind a map.
__device__ __forceinline__ float in_range(float p) {
  const int32_t bits = __float_as_int(p);
  return __int_as_float(max(bits, 1) | (bits & INT32_MIN));
}
__device__ __forceinline__ float joined(float p, float q) {
  const int32_t either = __float_as_int(p) | __float_as_int(q);
  return __int_as_float(max(__float_as_int(p * q), 1) | (either & INT32_MIN));
}
__device__ __forceinline__ float mapped(float p, float h, float u) {
  return __float_as_int(p) < 0 ? u : fmaf(p, h, u);
}
// Whether one of a chunk's factors is 0, from the least of their bits: a token
// costs half an instruction, whatever the gates are.  Looking at the factors only
// where their product is 0 takes the same without such gates, and 86 us for 59
// (8 x 4096 x 1024 bf16 forward) where one in a thousand forgets.
struct Least {
  uint32_t bits = ~0u;
  __device__ __forceinline__ void add(float a) { bits = min(bits, __float_as_uint(a)); }
  __device__ __forceinline__ float marked(float p) const {
    return bits == 0u ? -1.0f : in_range(p);
  }
};

// A thread's place: its strip and channels.
struct Place {
  int group;      // strip of the block
  uint32_t col;   // first channel
  uint32_t lane;  // among the lanes across the channels
  bool inside;    // the channels exist
  int32_t lo, hi; // tokens
  __device__ __forceinline__ Place(const Tokens &c, int V, int64_t block, uint32_t slice) {
    lane = threadIdx.x & ((1u << c.lane_bits) - 1u);
    group = static_cast<int>(threadIdx.x >> c.lane_bits);
    col = ((slice << c.lane_bits) + lane) * V;
    inside = col < c.width;
    const int32_t end = static_cast<int32_t>(min((block + 1) * c.block, c.n));
    lo = static_cast<int32_t>(
        min(block * c.block + static_cast<int64_t>(group) * c.strip, static_cast<int64_t>(end)));
    hi = min(lo + c.strip, end);
  }
};

// Rows of a strip: a wave's strips lie `strip` tokens apart, so the address of
// step k is a scalar that moves with k and a 32-bit offset per lane that does
// not.
template <typename T, int V>
struct Rows {
  using Global = __attribute__((address_space(1))) char *;
  using Word = typename std::conditional<sizeof(T) * V == 4, uint32_t, uint16_t>::type;
  Global base;       // of step 0, wave-uniform
  int64_t pitch;     // bytes per step, negative in reverse
  uint32_t offset;
  __device__ __forceinline__ Rows(const T *p, int64_t stride, const Tokens &c, const Place &at,
                                  int64_t block) {
    const int per_wave = 64 >> c.lane_bits;
    const int first = static_cast<int>(wave_index()) * per_wave, mine = at.group - first;
    const int64_t row_bytes = stride * static_cast<int64_t>(sizeof(T));
    const int64_t t0 = block * c.block + static_cast<int64_t>(first) * c.strip;
    const uint32_t step = static_cast<uint32_t>(c.strip * row_bytes);
    const uint32_t col = min(at.col, c.width - V) * static_cast<uint32_t>(sizeof(T));
    if (c.reverse) {
      base = (Global)p + (c.n - 1 - t0 - static_cast<int64_t>(per_wave - 1) * c.strip) * row_bytes;
      pitch = -row_bytes;
      offset = static_cast<uint32_t>(per_wave - 1 - mine) * step + col;
    } else {
      base = (Global)p + t0 * row_bytes;
      pitch = row_bytes;
      offset = static_cast<uint32_t>(mine) * step + col;
    }
  }
  // Step k's address without the lane's part, kept in scalar registers.
  __device__ __forceinline__ Global step(int64_t k) const {
    Global s = base + k * pitch;
    asm("" : "+s"(s));
    return s;
  }
  // The lane's offset, known to be 32 bits wide where it is added (else the
  // address is a 64-bit vector sum).
  __device__ __forceinline__ uint32_t lane_offset() const {
    uint32_t o = offset;
    asm("" : "+v"(o));
    return o;
  }
  __device__ __forceinline__ Word load(Global s, uint32_t o) const {
    return *(const __attribute__((address_space(1))) Word *)(s + o);
  }
  __device__ __forceinline__ void store(Global s, uint32_t o, Word x) const {
    *(__attribute__((address_space(1))) Word *)(s + o) = x;
  }
  __device__ __forceinline__ Word load(int64_t k) const { return load(step(k), lane_offset()); }
  __device__ __forceinline__ void store(int64_t k, Word x) const {
    store(step(k), lane_offset(), x);
  }
  // Element v of a word.
  static __device__ __forceinline__ float value(Word x, int v) {
    return static_cast<float>(__builtin_bit_cast(Pack<T, V>, x).v[v]);
  }
};

// kChunk rows from step j on, of which this lane has `count` in all; 0 past
// them.
template <typename R, typename Word>
__device__ __forceinline__ void load_chunk(const R &r, int32_t j, int32_t count,
                                           Word (&x)[kChunk]) {
  typename R::Global s = r.step(j);
  const uint32_t o = r.lane_offset();
  if (__all(j + kChunk <= count)) {
#pragma unroll
    for (int k = 0; k < kChunk; ++k) {
      x[k] = r.load(s, o);
      s += r.pitch;
      asm("" : "+s"(s));
    }
  } else {
#pragma unroll
    for (int k = 0; k < kChunk; ++k) x[k] = j + k < count ? r.load(j + k) : Word(0);
  }
}
template <typename R, typename T, int V>
__device__ __forceinline__ void store_chunk(const R &r, int32_t j,
                                            const Pack<T, V> (&x)[kChunk]) {
  typename R::Global s = r.step(j);
  const uint32_t o = r.lane_offset();
#pragma unroll
  for (int k = 0; k < kChunk; ++k) {
    r.store(s, o, __builtin_bit_cast(typename R::Word, x[k]));
    s += r.pitch;
    asm("" : "+s"(s));
  }
}

// The sequence that a walk is in: its number and tokens [first, last].
struct Cursor {
  int32_t s, first, last;

  // The sequence of token t; none (s = -1) where there is no such token.
  __device__ __forceinline__ void seek(const Tokens &c, int32_t t, bool some) {
    s = -1;
    first = last = -1;
    if (c.offsets == nullptr) {
      if (!some) return;
      s = static_cast<int32_t>(static_cast<uint32_t>(t) / static_cast<uint32_t>(c.length));
    } else {
      // The last sequence that starts at or before t, by the lanes of the
      // group together: 2^lane_bits probes a round.
      const uint32_t lanes = 1u << c.lane_bits, lane = lane_id() & (lanes - 1u);
      const uint32_t shift = lane_id() & ~(lanes - 1u);
      const uint64_t mask = lanes == 64u ? ~0ull : ((1ull << lanes) - 1ull);
      uint32_t lo = 0, hi = static_cast<uint32_t>(c.sequences);
      while (__any(hi - lo > 1)) {
        const uint32_t step = (hi - lo - 1) / (lanes + 1) + 1;
        const uint64_t q = lo + (static_cast<uint64_t>(lane) + 1) * step;
        const uint64_t under =
            ballot(q < hi && c.start(static_cast<int64_t>(q)) <= t) >> shift & mask;
        const uint32_t k = static_cast<uint32_t>(__popcll(under));
        hi = static_cast<uint32_t>(
            min(static_cast<uint64_t>(hi), lo + (static_cast<uint64_t>(k) + 1) * step));
        lo += k * step;
        if (hi <= lo) hi = lo + 1;  // offsets that do not ascend
      }
      if (!some) return;
      s = static_cast<int32_t>(lo);
    }
    bounds(c);
  }
  __device__ __forceinline__ void bounds(const Tokens &c) {
    first = static_cast<int32_t>(c.start(s));
    last = static_cast<int32_t>(c.start(s + 1) - 1);
  }
  // The sequences with a token that follow, and those before.
  __device__ __forceinline__ void next(const Tokens &c, int32_t t) {
    do {
      ++s;
      if (s >= c.sequences) {
        s = -1;
        first = last = -1;
        return;
      }
      bounds(c);
    } while (last < t);
  }
  __device__ __forceinline__ void previous(const Tokens &c, int32_t t) {
    do {
      --s;
      if (s < 0) {
        first = last = -1;
        return;
      }
      bounds(c);
    } while (first > t);
  }
};

// Whether tokens [t, t + kChunk) of every lane of the wave lie inside one
// sequence, and none but its first token is not a sequence's first (forward)
// or none is its last (backward).
__device__ __forceinline__ bool plain_forward(const Cursor &q, int32_t t, int32_t hi) {
  return __all(t + kChunk <= hi && t > q.first && t + kChunk - 1 <= q.last);
}
__device__ __forceinline__ bool plain_backward(const Cursor &q, int32_t t, int32_t hi) {
  return __all(t + kChunk <= hi && t > q.first && t + kChunk - 1 < q.last);
}

// The sequences of a chunk's tokens, and which are a sequence's first or last.
struct Marks {
  int32_t s[kChunk];
  uint32_t first, last;  // a bit for each
  __device__ __forceinline__ bool is_first(int k) const { return first >> k & 1u; }
  __device__ __forceinline__ bool is_last(int k) const { return last >> k & 1u; }
};

// The marks of tokens [t, t + kChunk), the lane's first `count` of which are
// there, from the sequence of a token at or before t (at or after the last one
// with kDown), which moves on to that of the chunk's far end.  The lanes of a
// group look at sixteen bounds or more together, one wait for all: 5000 x 128
// bf16 tokens of 1000 sequences, forward and back, 95 us, and 118 us token
// after token.
template <bool kDown>
__device__ __forceinline__ void find_marks(const Tokens &c, Cursor &q, int32_t t, int32_t count,
                                           Marks &m) {
  const uint32_t lanes = 1u << c.lane_bits, lane = lane_id() & (lanes - 1u);
  const uint32_t shift = lane_id() & ~(lanes - 1u);
  const uint64_t mask = lanes == 64u ? ~0ull : (1ull << lanes) - 1ull;
  constexpr int32_t kNone = kDown ? INT32_MIN : INT32_MAX;
  m.first = m.last = 0;
#pragma unroll
  for (int k = 0; k < kChunk; ++k) {
    m.s[k] = q.s;
    if (t + k == q.first) m.first |= 1u << k;
    if (t + k == q.last) m.last |= 1u << k;
  }
  int32_t end = kNone;  // the farthest bound looked at
  for (uint32_t i = 0; i < 16; i += lanes) {
    const int64_t at = kDown ? int64_t{q.s} - lane - i : int64_t{q.s} + 1 + lane + i;
    const bool some = q.s >= 0 && at >= 0 && at <= c.sequences;
    const int32_t b = some ? static_cast<int32_t>(c.start(at)) : kNone;
#pragma unroll
    for (int k = 0; k < kChunk; ++k) {
      const uint64_t past = ballot(kDown ? b > t + k : b <= t + k) >> shift & mask;
      m.s[k] += (kDown ? -1 : 1) * __popcll(past);
      if (ballot(b == t + k) >> shift & mask) m.first |= 1u << k;
      if (ballot(b == t + k + 1) >> shift & mask) m.last |= 1u << k;
    }
    end = __shfl(b, static_cast<int>(shift + lanes - 1u), 64);
  }
  if (__any(q.s >= 0 && count > 0 && (kDown ? end > t : end <= t + kChunk))) {
    // More bounds than that: sequences without a token.
    m.first = m.last = 0;
    Cursor w = q;
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      const int k = kDown ? kChunk - 1 - i : i;
      if (k < count) {
        if (kDown && t + k < w.first) w.previous(c, t + k);
        if (!kDown && t + k > w.last) w.next(c, t + k);
        m.s[k] = w.s;
        if (t + k == w.first) m.first |= 1u << k;
        if (t + k == w.last) m.last |= 1u << k;
      }
    }
    q = w;
    return;
  }
  // Offsets that do not cover the tokens: nothing to mark there.
#pragma unroll
  for (int k = 0; k < kChunk; ++k) {
    if (m.s[k] < 0 || m.s[k] >= c.sequences) {
      m.s[k] = -1;
      m.first &= ~(1u << k);
      m.last &= ~(1u << k);
    }
  }
  const int32_t s = m.s[kDown ? 0 : kChunk - 1];
  if (s != q.s) {
    q.s = s;
    q.first = q.last = -1;
    if (s >= 0) q.bounds(c);
  }
}

template <int V>
__device__ __forceinline__ void load_state(const float *p, const Tokens &c, const Place &at,
                                           int64_t s, float (&h)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v)
    h[v] = p != nullptr && at.inside ? p[c.state_row(s) * c.width + at.col + v] : 0.0f;
}

// ------------------------------------------------------------- forward ---

// The map of the strip: p, u.
template <typename T, int V>
__device__ __forceinline__ void compose_forward(const Rows<T, V> &xr, const Rows<T, V> &gr,
                                                const float *initial, const Tokens &c,
                                                const Place &at, float (&p)[V], float (&u)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) p[v] = 1.0f, u[v] = 0.0f;
  Cursor q;
  q.seek(c, at.lo, at.lo < at.hi);
  const int32_t count = at.hi - at.lo;
  using R = Rows<T, V>;
  typename R::Word x[kChunk], g[kChunk];
  for (int32_t j = 0; __any(j < count); j += kChunk) {
    const int32_t t = at.lo + j;
    load_chunk(xr, j, count, x);
    load_chunk(gr, j, count, g);
    if (plain_forward(q, t, at.hi)) {
      float p1[V], u1[V];
      Least least[V];
#pragma unroll
      for (int v = 0; v < V; ++v) p1[v] = p[v], u1[v] = u[v];
#pragma unroll
      for (int k = 0; k < kChunk; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float a, b;
          gate_pair(R::value(g[k], v), a, b);
          u1[v] = fmaf(a, u1[v], b * R::value(x[k], v));
          p1[v] *= a;
          least[v].add(a);
        }
      bool fine = true;
#pragma unroll
      for (int v = 0; v < V; ++v) fine = fine && finite(u1[v]) && finite(p1[v]);
      if (__all(fine)) {
#pragma unroll
        for (int v = 0; v < V; ++v) p[v] = least[v].marked(p1[v]), u[v] = u1[v];
        continue;
      }
      // Loaded again rather than held through the form above.
      load_chunk(xr, j, count, x);
      load_chunk(gr, j, count, g);
    }
    Marks m;
    find_marks<false>(c, q, t, count - j, m);
#pragma unroll
    for (int k = 0; k < kChunk; ++k) {
      if (j + k < count) {
        const bool first = m.is_first(k);
        float h0[V];
        if (first) load_state<V>(initial, c, at, m.s[k], h0);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float a, b;
          gate_pair(R::value(g[k], v), a, b);
          const float fresh = scaled<true>(b, R::value(x[k], v));
          u[v] = applied<true>(a, first ? h0[v] : u[v], fresh);
          p[v] = first || a == 0.0f ? -1.0f : p[v] * a;
        }
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] = in_range(p[v]);
  }
}

// The states of the strip from h, the one before it.  kept: the state before
// each kChunk tokens (may be null).
template <typename T, int V>
__device__ __forceinline__ void walk_forward(const Rows<T, V> &xr, const Rows<T, V> &gr,
                                             const Rows<T, V> &yr, const float *initial,
                                             const Tokens &c, const Place &at, float *kept,
                                             float *final, float (&h)[V]) {
  Cursor q;
  q.seek(c, at.lo, at.lo < at.hi);
  const int32_t count = at.hi - at.lo;
  using R = Rows<T, V>;
  typename R::Word x[kChunk], g[kChunk];
  for (int32_t j = 0; __any(j < count); j += kChunk) {
    const int32_t t = at.lo + j;
    load_chunk(xr, j, count, x);
    load_chunk(gr, j, count, g);
    if (kept != nullptr && j < count && at.inside) {
#pragma unroll
      for (int v = 0; v < V; ++v) kept[static_cast<int64_t>(j / kChunk) * c.width + v] = h[v];
    }
    // A sequence's last token stores its state: not in the plain form.
    if (plain_backward(q, t, at.hi)) {
      float h1[V];
      Pack<T, V> y[kChunk];
#pragma unroll
      for (int v = 0; v < V; ++v) h1[v] = h[v];
#pragma unroll
      for (int k = 0; k < kChunk; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float a, b;
          gate_pair(R::value(g[k], v), a, b);
          h1[v] = fmaf(a, h1[v], b * R::value(x[k], v));
          y[k].v[v] = static_cast<T>(h1[v]);
        }
      bool fine = true;
#pragma unroll
      for (int v = 0; v < V; ++v) fine = fine && finite(h1[v]);
      if (__all(fine)) {
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = h1[v];
        if (at.inside) store_chunk(yr, j, y);
        continue;
      }
      load_chunk(xr, j, count, x);
      load_chunk(gr, j, count, g);
    }
    Marks m;
    find_marks<false>(c, q, t, count - j, m);
#pragma unroll
    for (int k = 0; k < kChunk; ++k) {
      if (j + k < count) {
        Pack<T, V> y;
        if (m.is_first(k)) load_state<V>(initial, c, at, m.s[k], h);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float a, b;
          gate_pair(R::value(g[k], v), a, b);
          h[v] = applied<true>(a, h[v], scaled<true>(b, R::value(x[k], v)));
          y.v[v] = static_cast<T>(h[v]);
        }
        if (at.inside) {
          yr.store(j + k, __builtin_bit_cast(typename R::Word, y));
          if (m.is_last(k)) {
#pragma unroll
            for (int v = 0; v < V; ++v) final[c.state_row(m.s[k]) * c.width + at.col + v] = h[v];
          }
        }
      }
    }
  }
}

// ------------------------------------------------------------ backward ---

// The backward map of the strip, from its last token to its first.
template <typename T, int V>
__device__ __forceinline__ void compose_backward(const Rows<T, V> &gr, const Rows<T, V> &vr,
                                                 const float *v_final, const Tokens &c,
                                                 const Place &at, float (&p)[V], float (&u)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) p[v] = 1.0f, u[v] = 0.0f;
  const int32_t count = at.hi - at.lo;
  Cursor q;
  q.seek(c, at.hi - 1, count > 0);
  using R = Rows<T, V>;
  typename R::Word g[kChunk], d[kChunk];
  for (int32_t j = c.steps - kChunk; j >= 0; j -= kChunk) {
    if (!__any(j < count)) continue;
    const int32_t t = at.lo + j;
    load_chunk(gr, j, count, g);
    load_chunk(vr, j, count, d);
    if (plain_backward(q, t, at.hi)) {
      float p1[V], u1[V];
      Least least[V];
#pragma unroll
      for (int v = 0; v < V; ++v) p1[v] = p[v], u1[v] = u[v];
#pragma unroll
      for (int k = kChunk - 1; k >= 0; --k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float a, b;
          gate_pair(R::value(g[k], v), a, b);
          u1[v] = a * (R::value(d[k], v) + u1[v]);
          p1[v] *= a;
          least[v].add(a);
        }
      bool fine = true;
#pragma unroll
      for (int v = 0; v < V; ++v) fine = fine && finite(u1[v]) && finite(p1[v]);
      if (__all(fine)) {
#pragma unroll
        for (int v = 0; v < V; ++v) p[v] = least[v].marked(p1[v]), u[v] = u1[v];
        continue;
      }
      load_chunk(gr, j, count, g);
      load_chunk(vr, j, count, d);
    }
    Marks m;
    find_marks<true>(c, q, t, count - j, m);
#pragma unroll
    for (int k = kChunk - 1; k >= 0; --k) {
      if (j + k < count) {
        const bool last = m.is_last(k);
        float f0[V];
        if (last) load_state<V>(v_final, c, at, m.s[k], f0);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float a, b;
          gate_pair(R::value(g[k], v), a, b);
          u[v] = scaled<true>(a, R::value(d[k], v) + (last ? f0[v] : u[v]));
          p[v] = last || a == 0.0f ? -1.0f : p[v] * a;
        }
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] = in_range(p[v]);
  }
}

// The gradients of the strip's tokens from f, the gradient that reaches the
// state after it.
template <typename T, int V>
__device__ __forceinline__ void walk_backward(const Rows<T, V> &xr, const Rows<T, V> &gr,
                                              const Rows<T, V> &vr, const Rows<T, V> &dxr,
                                              const Rows<T, V> &dgr, const float *initial,
                                              const float *v_final, const Tokens &c,
                                              const Place &at, const float *kept,
                                              float *v_initial, float *s_before,
                                              float (&f)[V]) {
  const int32_t count = at.hi - at.lo;
  Cursor q;
  q.seek(c, at.hi - 1, count > 0);
  using R = Rows<T, V>;
  typename R::Word x[kChunk], g[kChunk], d[kChunk];
  for (int32_t j = c.steps - kChunk; j >= 0; j -= kChunk) {
    if (!__any(j < count)) continue;
    const int32_t t = at.lo + j;
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v)
      h[v] = j < count && at.inside ? kept[static_cast<int64_t>(j / kChunk) * c.width + v] : 0.0f;
    load_chunk(xr, j, count, x);
    load_chunk(gr, j, count, g);
    load_chunk(vr, j, count, d);
    if (plain_backward(q, t, at.hi)) {
      float prior[kChunk][V], a[kChunk][V], b[kChunk][V], f1[V], h1[V];
#pragma unroll
      for (int v = 0; v < V; ++v) f1[v] = f[v], h1[v] = h[v];
#pragma unroll
      for (int k = 0; k < kChunk; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          gate_pair(R::value(g[k], v), a[k][v], b[k][v]);
          const float xv = R::value(x[k], v);
          prior[k][v] = h1[v] - xv;
          h1[v] = fmaf(a[k][v], h1[v], b[k][v] * xv);
        }
      // Stored as they come; where the chunk turns out not to be finite, the
      // other form stores again.
#pragma unroll
      for (int k = kChunk - 1; k >= 0; --k) {
        Pack<T, V> dx, dg;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float gk = R::value(d[k], v) + f1[v], vx = b[k][v] * gk;
          f1[v] = a[k][v] * gk;
          dx.v[v] = static_cast<T>(vx);
          dg.v[v] = static_cast<T>(a[k][v] * (vx * prior[k][v]));
        }
        if (at.inside) {
          dxr.store(j + k, __builtin_bit_cast(typename R::Word, dx));
          dgr.store(j + k, __builtin_bit_cast(typename R::Word, dg));
        }
      }
      bool fine = true;
#pragma unroll
      for (int v = 0; v < V; ++v) fine = fine && finite(f1[v]) && finite(h1[v]);
      if (__all(fine)) {
#pragma unroll
        for (int v = 0; v < V; ++v) f[v] = f1[v];
        continue;
      }
      load_chunk(xr, j, count, x);
      load_chunk(gr, j, count, g);
      load_chunk(vr, j, count, d);
    }
    // Token by token: the states before them first (in LDS, so that the other
    // form keeps its registers), then back.
    Marks m;
    find_marks<true>(c, q, t, count - j, m);
#pragma unroll
    for (int k = 0; k < kChunk; ++k) {
      if (j + k < count) {
        if (m.is_first(k)) load_state<V>(initial, c, at, m.s[k], h);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float a, b;
          gate_pair(R::value(g[k], v), a, b);
          s_before[(k * V + v) * kThreads + threadIdx.x] = h[v];
          h[v] = applied<true>(a, h[v], scaled<true>(b, R::value(x[k], v)));
        }
      }
    }
#pragma unroll
    for (int k = kChunk - 1; k >= 0; --k) {
      if (j + k < count) {
        Pack<T, V> dx, dg;
        if (m.is_last(k)) load_state<V>(v_final, c, at, m.s[k], f);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float a, b;
          gate_pair(R::value(g[k], v), a, b);
          const float gk = R::value(d[k], v) + f[v], vx = scaled<true>(b, gk);
          const float before = s_before[(k * V + v) * kThreads + threadIdx.x];
          const float vg = a * (vx * (before - R::value(x[k], v)));
          dx.v[v] = static_cast<T>(vx);
          dg.v[v] = static_cast<T>(a == 0.0f || b == 0.0f ? 0.0f : vg);
          f[v] = scaled<true>(a, gk);
        }
        if (at.inside) {
          dxr.store(j + k, __builtin_bit_cast(typename R::Word, dx));
          dgr.store(j + k, __builtin_bit_cast(typename R::Word, dg));
          if (m.is_first(k) && v_initial != nullptr) {
#pragma unroll
            for (int v = 0; v < V; ++v)
              v_initial[c.state_row(m.s[k]) * c.width + at.col + v] = f[v];
          }
        }
      }
    }
  }
}

// --------------------------------------------------- maps between strips ---

// The strips' maps of a block in LDS, as [group][lane] of V (p, u) pairs.
template <int V>
__device__ __forceinline__ void put_map(float *s_map, const float (&p)[V], const float (&u)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s_map[(threadIdx.x * V + v) * 2] = p[v];
    s_map[(threadIdx.x * V + v) * 2 + 1] = u[v];
  }
}

// The maps that a packed call keeps between its launches: of every strip,
// strips [n][width] of (p, u), and of every block of strips, likewise.
template <int V>
__device__ __forceinline__ void store_map(float *maps, int64_t row, const Tokens &c,
                                          const Place &at, const float (&p)[V],
                                          const float (&u)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float *m = maps + (row * c.width + at.col + v) * 2;
    m[0] = p[v];
    m[1] = u[v];
  }
}

// Blocks that share rows' cache lines (slices of one block of tokens) run on
// one XCD.
__device__ __forceinline__ void block_and_slice(uint32_t slices, int64_t &block,
                                                uint32_t &slice) {
  const uint32_t id = xcd_swizzle(blockIdx.x, gridDim.x);
  block = id / slices;
  slice = id - static_cast<uint32_t>(block) * slices;
}

// The maps of the strips and of each block of them.  500k x 64 bf16: 35 us, the
// tokens' 128 MB at 3.7 TB/s; 200k x 99 f32: 58 us forward and 37 back for 158 MB,
// of which 184 and 189 MB are read (see scan_bwd_kernel).
template <typename T, int V, bool kBack>
__global__ __launch_bounds__(kThreads) void scan_maps_kernel(
    const T *__restrict__ a, int64_t a_stride, const T *__restrict__ b, int64_t b_stride,
    const float *__restrict__ state, Tokens c, uint32_t slices, float *__restrict__ strips,
    float *__restrict__ blocks) {
  extern __shared__ float s_map[];
  int64_t block;
  uint32_t slice;
  block_and_slice(slices, block, slice);
  const int groups = kThreads >> c.lane_bits;
  const Place at(c, V, block, slice);
  const Rows<T, V> ar(a, a_stride, c, at, block), br(b, b_stride, c, at, block);
  float p[V], u[V];
  if constexpr (kBack)
    compose_backward<T, V>(ar, br, state, c, at, p, u);
  else
    compose_forward<T, V>(ar, br, state, c, at, p, u);
  put_map<V>(s_map, p, u);
  if (at.inside)
    store_map<V>(strips, block * groups + at.group, c, at, p, u);
  __syncthreads();
  // The block's map: everything from its far end, composed by one group.
  if (at.group != (kBack ? groups - 1 : 0) || !at.inside) return;
  for (int i = 1; i < groups; ++i) {
    const int q = kBack ? groups - 1 - i : i;
    const float *m = s_map + ((q << c.lane_bits) + static_cast<int>(at.lane)) * V * 2;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      u[v] = mapped(m[v * 2], u[v], m[v * 2 + 1]);
      p[v] = joined(p[v], m[v * 2]);
    }
  }
  store_map<V>(blocks, block, c, at, p, u);
}

// Sequences without a token: the state they end in (or its gradient) is the
// one they began with.
__device__ __forceinline__ void empty_state(const Tokens &c, int64_t i, const float *in,
                                            float *out) {
  const int64_t s = i / c.width;
  if (s >= c.sequences || (c.offsets != nullptr && c.offsets[s] < c.offsets[s + 1])) return;
  out[i] = in != nullptr ? in[i] : 0.0f;
}

// The state that enters each block, from the blocks' maps in order (from the
// last block down with `down`).  A launch block takes kCarryCols channels, and
// kCarryRows x kCarryPer maps of each at a time: a thread composes kCarryPer of
// them in registers, the rows of a wave meet by lane shifts, the waves in LDS.
// Launch blocks past the channels' look after the sequences without a token.
// 5 us with 489 to 977 blocks' maps, most of it the launch and two waits.
constexpr int kCarryCols = 4, kCarryRows = 1024 / kCarryCols, kCarryPer = 4;
__global__ __launch_bounds__(1024) void scan_carry_kernel(const float2 *__restrict__ maps,
                                                          int32_t blocks, Tokens c, int32_t down,
                                                          uint32_t channel_blocks,
                                                          float *__restrict__ carries,
                                                          const float *__restrict__ empty_in,
                                                          float *__restrict__ empty_out) {
  if (blockIdx.x >= channel_blocks) {
    empty_state(c, static_cast<int64_t>(blockIdx.x - channel_blocks) * 1024 + threadIdx.x,
                empty_in, empty_out);
    return;
  }
  __shared__ float2 s_map[16][kCarryCols];
  const uint32_t lane = threadIdx.x % kCarryCols, wave = threadIdx.x / 64;
  const int32_t row = static_cast<int32_t>(threadIdx.x / kCarryCols);
  const uint32_t col = min(blockIdx.x * kCarryCols + lane, c.width - 1);
  const bool inside = blockIdx.x * kCarryCols + lane < c.width;
  float h = 0.0f;  // the state that enters the round
  for (int32_t r0 = 0; r0 < blocks; r0 += kCarryRows * kCarryPer) {
    const int32_t i0 = r0 + row * kCarryPer;
    float2 m[kCarryPer];
#pragma unroll
    for (int k = 0; k < kCarryPer; ++k) {
      const int32_t i = min(i0 + k, blocks - 1);
      m[k] = maps[static_cast<int64_t>(down ? blocks - 1 - i : i) * c.width + col];
    }
    float p = 1.0f, u = 0.0f;
#pragma unroll
    for (int k = 0; k < kCarryPer; ++k) {
      if (i0 + k >= blocks) m[k] = make_float2(1.0f, 0.0f);
      u = mapped(m[k].x, u, m[k].y);
      p = joined(p, m[k].x);
    }
#pragma unroll
    for (int off = kCarryCols; off < 64; off *= 2) {
      const float pb = __shfl_up(p, off, 64), ub = __shfl_up(u, off, 64);
      if (static_cast<int>(threadIdx.x % 64) >= off) {
        u = mapped(p, ub, u);
        p = joined(p, pb);
      }
    }
    if (threadIdx.x % 64 >= 64 - kCarryCols) s_map[wave][lane] = make_float2(p, u);
    float before_p = __shfl_up(p, kCarryCols, 64), before_u = __shfl_up(u, kCarryCols, 64);
    if (threadIdx.x % 64 < kCarryCols) before_p = 1.0f, before_u = 0.0f;
    __syncthreads();
    float mine = h;
#pragma unroll
    for (uint32_t w = 0; w < 16; ++w) {
      if (w == wave) mine = h;
      h = mapped(s_map[w][lane].x, h, s_map[w][lane].y);
    }
    __syncthreads();
    mine = mapped(before_p, mine, before_u);
#pragma unroll
    for (int k = 0; k < kCarryPer; ++k) {
      const int32_t i = i0 + k;
      if (inside && i < blocks)
        carries[static_cast<int64_t>(down ? blocks - 1 - i : i) * c.width + col] = mine;
      mine = mapped(m[k].x, mine, m[k].y);
    }
  }
}

// The state that enters the thread's strip in a packed call: the block's,
// through the maps of the block's strips before.
template <int V, bool kDown>
__device__ __forceinline__ void enter_strip(const float *strips, const float *carries,
                                            const Tokens &c, const Place &at, int groups,
                                            int64_t block, float (&h)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = at.inside ? carries[block * c.width + at.col + v] : 0.0f;
  if (!at.inside) return;
  const int count = kDown ? groups - 1 - at.group : at.group;
  for (int i = 0; i < count; ++i) {
    const int q = kDown ? groups - 1 - i : i;
    const float *m = strips + ((block * groups + q) * c.width + at.col) * 2;
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = mapped(m[v * 2], h[v], m[v * 2 + 1]);
  }
}

// How a walk gets the state that enters its strip.
enum Mode { kPacked, kRounds, kOwn };

// The states, each walk from the one that enters its strip; kept
// [strips][steps / kChunk][width].  500k x 64 bf16: 34 us, 192 MB at 5.6 TB/s, the
// tokens' second reading from the last-level cache.
template <typename T, int V, int kMode>
__global__ __launch_bounds__(kThreads) void scan_fwd_kernel(
    const T *__restrict__ x, int64_t x_stride, const T *__restrict__ gate, int64_t g_stride,
    const float *__restrict__ initial, Tokens c, uint32_t slices,
    const float *__restrict__ strips, const float *__restrict__ carries, float *__restrict__ kept,
    T *__restrict__ y, float *__restrict__ final) {
  int64_t block;
  uint32_t slice;
  block_and_slice(slices, block, slice);
  const int groups = kThreads >> c.lane_bits;
  const Place at(c, V, block, slice);
  const Rows<T, V> xr(x, x_stride, c, at, block), gr(gate, g_stride, c, at, block);
  const Rows<T, V> yr(y, c.width, c, at, block);
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = 0.0f;
  if constexpr (kMode == kPacked) {
    enter_strip<V, false>(strips, carries, c, at, groups, block, h);
  }
  if (kept != nullptr)
    kept += (block * groups + at.group) * (c.steps / kChunk) * c.width + at.col;
  walk_forward<T, V>(xr, gr, yr, initial, c, at, kept, final, h);
}

// The gradients, likewise.  200k x 99 f32: 105 us, 535 MB at 5.1 TB/s, bound by
// bytes, a quarter of which nobody needs: a row of 396 bytes is two blocks' slices,
// and both fetch (and write parts of) the cache lines between them, 351 MB for
// the 248 of operands and kept states and 184 for the 158 of gradients.
template <typename T, int V, int kMode>
__global__ __launch_bounds__(kThreads) void scan_bwd_kernel(
    const T *__restrict__ x, int64_t x_stride, const T *__restrict__ gate, int64_t g_stride,
    const float *__restrict__ initial, const T *__restrict__ v_y, int64_t v_stride,
    const float *__restrict__ v_final, Tokens c, uint32_t slices,
    const float *__restrict__ strips, const float *__restrict__ carries,
    const float *__restrict__ kept, T *__restrict__ v_x, T *__restrict__ v_gate,
    float *__restrict__ v_initial) {
  __shared__ float s_before[kThreads * V * kChunk];
  int64_t block;
  uint32_t slice;
  block_and_slice(slices, block, slice);
  const int groups = kThreads >> c.lane_bits;
  const Place at(c, V, block, slice);
  const Rows<T, V> xr(x, x_stride, c, at, block), gr(gate, g_stride, c, at, block);
  const Rows<T, V> vr(v_y, v_stride, c, at, block);
  const Rows<T, V> dxr(v_x, c.width, c, at, block), dgr(v_gate, c.width, c, at, block);
  float f[V];
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = 0.0f;
  if constexpr (kMode == kPacked) {
    enter_strip<V, true>(strips, carries, c, at, groups, block, f);
  }
  kept += (block * groups + at.group) * (c.steps / kChunk) * c.width + at.col;
  walk_backward<T, V>(xr, gr, vr, dxr, dgr, initial, v_final, c, at, kept, v_initial, s_before,
                      f);
}

// ------------------------------------------------- whole sequences at once ---

// A block whose tokens are whole sequences walks them in rounds: its groups
// take kChunk tokens each, side by side, and the state that leaves the last one
// enters the next round.  So x and gate are read once, and a round's words are
// on their way while the one before is worked on.  32 x 1024 x 1024 bf16 takes
// 55 us forward (201 MB, 3.7 TB/s) and 77 us back (344 MB, 4.5 TB/s); with one
// block of 8 waves per CU and 64 bytes of a row (8 x 4096 x 1024) 70 and 98 us,
// where a round's chain of waits bounds it (for words, for the stores of the round
// before, which the same counter holds, and for the other waves' maps): the
// vector units are busy a third of the time.  The packed form takes 185 us for
// the latter, its second reading of the tokens included.

// What a block's round leaves in LDS: the maps of its waves' tokens.
template <int V>
struct Rounds {
  alignas(16) float map[2][kRoundThreads / 64][32][2 * V];
};

// Chunks of a block of whole sequences.
__device__ __forceinline__ int64_t block_chunks(const Tokens &c) {
  return (c.block + kChunk - 1) / kChunk;
}

// The lane's place reaches to the block's end; the block's tokens.
__device__ __forceinline__ int32_t round_place(const Tokens &c, int64_t block, Place &at) {
  const int64_t end = min((block + 1) * c.block, c.n);
  at.hi = static_cast<int32_t>(end);
  return static_cast<int32_t>(end - block * c.block);
}

// A round's words on their way to LDS, each lane's to a place of its own: held
// in registers until the next round, the compiler waits for them where paths
// meet.  words [k][threads] from `at` on; a lane without a token keeps what is
// there.
template <typename R>
__device__ __forceinline__ void fetch_chunk(const R &r, int32_t j, int32_t count,
                                            uint32_t *words) {
  typename R::Global s = r.step(j);
  const uint32_t o = r.lane_offset();
  words += wave_index() * 64;
  const bool all = __all(j + kChunk <= count);
#pragma unroll
  for (int k = 0; k < kChunk; ++k) {
    if (all || j + k < count) {
      const auto *from = (const __attribute__((address_space(1))) void *)(s + o);
      auto *to = (__attribute__((address_space(3))) void *)(words + k * kRoundThreads);
      if constexpr (sizeof(typename R::Word) == 4)
        __builtin_amdgcn_global_load_lds(from, to, 4, 0, 0);
      else
        __builtin_amdgcn_global_load_lds(from, to, 2, 0, 0);
    }
    s += r.pitch;
    asm("" : "+s"(s));
  }
}
template <typename Word>
__device__ __forceinline__ void take_chunk(const uint32_t *words, Word (&x)[kChunk]) {
#pragma unroll
  for (int k = 0; k < kChunk; ++k) x[k] = static_cast<Word>(words[k * kRoundThreads + threadIdx.x]);
}
// The words fetched for this round have arrived (and the stores of the round before
// are done: one counter holds both); those taken may be replaced.
__device__ __forceinline__ void words_arrived() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}
__device__ __forceinline__ void words_taken() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// From the maps of the lanes' chunks to the state that enters each: through
// the wave's groups by lane shifts and through the waves in LDS, from `carry`,
// the state that enters the round, which becomes the one that leaves it.
// Backwards with kDown.
template <int V, bool kDown>
__device__ __forceinline__ void enter_chunk(Rounds<V> &s, int turn, const Tokens &c,
                                            const Place &at, float (&p)[V], float (&u)[V],
                                            float (&carry)[V], float (&h)[V]) {
  const int lanes = 1 << c.lane_bits, id = static_cast<int>(lane_id());
  const int ahead = kDown ? 63 - id : id;  // lanes before this one
  for (int off = lanes; off < 64; off *= 2) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float pb = kDown ? __shfl_down(p[v], off, 64) : __shfl_up(p[v], off, 64);
      const float ub = kDown ? __shfl_down(u[v], off, 64) : __shfl_up(u[v], off, 64);
      if (ahead >= off) {
        u[v] = mapped(p[v], ub, u[v]);
        p[v] = joined(p[v], pb);
      }
    }
  }
  const int wave = static_cast<int>(wave_index()), waves = static_cast<int>(blockDim.x / 64);
  if (ahead >= 64 - lanes) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s.map[turn][wave][at.lane][2 * v] = p[v];
      s.map[turn][wave][at.lane][2 * v + 1] = u[v];
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    p[v] = kDown ? __shfl_down(p[v], lanes, 64) : __shfl_up(p[v], lanes, 64);
    u[v] = kDown ? __shfl_down(u[v], lanes, 64) : __shfl_up(u[v], lanes, 64);
    if (ahead < lanes) p[v] = 1.0f, u[v] = 0.0f;
  }
  // Not __syncthreads, which would also wait for the words on their way.
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll 4
  for (int i = 0; i < waves; ++i) {
    const int w = kDown ? waves - 1 - i : i;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (w == wave) h[v] = carry[v];
      carry[v] = mapped(s.map[turn][w][at.lane][2 * v], carry[v],
                        s.map[turn][w][at.lane][2 * v + 1]);
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = mapped(p[v], h[v], u[v]);
}

// kept [blocks][chunks of a block][width].
template <typename T, int V>
__global__ __launch_bounds__(kRoundThreads) void scan_fwd_rounds_kernel(
    const T *__restrict__ tokens, int64_t x_stride, const T *__restrict__ gate, int64_t g_stride,
    const float *__restrict__ initial, Tokens c, uint32_t slices, float *__restrict__ kept,
    T *__restrict__ y, float *__restrict__ final) {
  __shared__ Rounds<V> s_rounds;
  __shared__ uint32_t s_words[2 * kChunk * kRoundThreads];  // x, gate
  int64_t block;
  uint32_t slice;
  block_and_slice(slices, block, slice);
  Place at(c, V, block, slice);
  const int32_t total = round_place(c, block, at), count = at.hi - at.lo;
  const int32_t span = static_cast<int32_t>(blockDim.x >> c.lane_bits) * kChunk;
  using R = Rows<T, V>;
  const R xr(tokens, x_stride, c, at, block), gr(gate, g_stride, c, at, block);
  const R yr(y, c.width, c, at, block);
  if (kept != nullptr)
    kept += (block * block_chunks(c) + at.group) * c.width + at.col;
  Cursor q;
  q.seek(c, at.lo, at.lo < at.hi);
  float carry[V];
#pragma unroll
  for (int v = 0; v < V; ++v) carry[v] = 0.0f;
  fetch_chunk(xr, 0, count, s_words);
  fetch_chunk(gr, 0, count, s_words + kChunk * kRoundThreads);
  int turn = 0;
  for (int32_t j = 0; j < total; j += span, turn ^= 1) {
    const int32_t t = at.lo + j;
    typename R::Word x[kChunk], g[kChunk];
    words_arrived();
    take_chunk(s_words, x);
    take_chunk(s_words + kChunk * kRoundThreads, g);
    if (j + span < total) {
      words_taken();
      fetch_chunk(xr, j + span, count, s_words);
      fetch_chunk(gr, j + span, count, s_words + kChunk * kRoundThreads);
    }
    float a[kChunk][V], fresh[kChunk][V], p[V], u[V], h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] = 1.0f, u[v] = 0.0f;
#pragma unroll
    for (int k = 0; k < kChunk; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float b;
        gate_pair(R::value(g[k], v), a[k][v], b);
        fresh[k][v] = scaled<true>(b, R::value(x[k], v));
      }
    const bool plain = plain_backward(q, t, at.hi);
    bool fine = plain;
    if (plain) {
      Least least[V];
#pragma unroll
      for (int k = 0; k < kChunk; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          u[v] = fmaf(a[k][v], u[v], fresh[k][v]);
          p[v] *= a[k][v];
          least[v].add(a[k][v]);
        }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        fine = fine && finite(u[v]) && finite(p[v]);
        p[v] = least[v].marked(p[v]);
      }
      fine = __all(fine);
    }
    if (!fine) {
#pragma unroll
      for (int v = 0; v < V; ++v) p[v] = 1.0f, u[v] = 0.0f;
      Cursor w = q;
#pragma unroll
      for (int k = 0; k < kChunk; ++k) {
        if (j + k < count) {
          if (t + k > w.last) w.next(c, t + k);
          const bool first = t + k == w.first;
          float h0[V];
          if (first) load_state<V>(initial, c, at, w.s, h0);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            u[v] = applied<true>(a[k][v], first ? h0[v] : u[v], fresh[k][v]);
            p[v] = first || a[k][v] == 0.0f ? -1.0f : p[v] * a[k][v];
          }
        }
      }
#pragma unroll
      for (int v = 0; v < V; ++v) p[v] = in_range(p[v]);
    }
    enter_chunk<V, false>(s_rounds, turn, c, at, p, u, carry, h);
    if (kept != nullptr && j < count && at.inside) {
#pragma unroll
      for (int v = 0; v < V; ++v) kept[static_cast<int64_t>(j / kChunk) * c.width + v] = h[v];
    }
    if (fine) {
      float h1[V];
      Pack<T, V> out[kChunk];
#pragma unroll
      for (int v = 0; v < V; ++v) h1[v] = h[v];
#pragma unroll
      for (int k = 0; k < kChunk; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          h1[v] = fmaf(a[k][v], h1[v], fresh[k][v]);
          out[k].v[v] = static_cast<T>(h1[v]);
        }
#pragma unroll
      for (int v = 0; v < V; ++v) fine = fine && finite(h1[v]);
      if (__all(fine)) {
        if (at.inside) store_chunk(yr, j, out);
        continue;
      }
    }
#pragma unroll
    for (int k = 0; k < kChunk; ++k) {
      if (j + k < count) {
        if (t + k > q.last) q.next(c, t + k);
        if (t + k == q.first) load_state<V>(initial, c, at, q.s, h);
        Pack<T, V> out;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          h[v] = applied<true>(a[k][v], h[v], fresh[k][v]);
          out.v[v] = static_cast<T>(h[v]);
        }
        if (at.inside) {
          yr.store(j + k, __builtin_bit_cast(typename R::Word, out));
          if (t + k == q.last) {
#pragma unroll
            for (int v = 0; v < V; ++v) final[c.state_row(q.s) * c.width + at.col + v] = h[v];
          }
        }
      }
    }
  }
}

template <typename T, int V>
__global__ __launch_bounds__(kRoundThreads) void scan_bwd_rounds_kernel(
    const T *__restrict__ tokens, int64_t x_stride, const T *__restrict__ gate, int64_t g_stride,
    const float *__restrict__ initial, const T *__restrict__ v_y, int64_t v_stride,
    const float *__restrict__ v_final, Tokens c, uint32_t slices,
    const float *__restrict__ kept, T *__restrict__ v_x, T *__restrict__ v_gate,
    float *__restrict__ v_initial) {
  __shared__ Rounds<V> s_rounds;
  __shared__ uint32_t s_words[(3 * kChunk + V) * kRoundThreads];  // x, gate, v_y, kept
  int64_t block;
  uint32_t slice;
  block_and_slice(slices, block, slice);
  Place at(c, V, block, slice);
  const int32_t total = round_place(c, block, at), count = at.hi - at.lo;
  const int32_t span = static_cast<int32_t>(blockDim.x >> c.lane_bits) * kChunk;
  using R = Rows<T, V>;
  const R xr(tokens, x_stride, c, at, block), gr(gate, g_stride, c, at, block);
  const R vr(v_y, v_stride, c, at, block);
  const R dxr(v_x, c.width, c, at, block), dgr(v_gate, c.width, c, at, block);
  kept += block * block_chunks(c) * c.width + min(at.col, c.width - V);
  const int32_t last_chunk = (total - 1) / kChunk;
  Cursor q;
  q.seek(c, at.hi - 1, total > 0);
  float carry[V];
#pragma unroll
  for (int v = 0; v < V; ++v) carry[v] = 0.0f;
  auto fetch = [&](int32_t j) {
    fetch_chunk(xr, j, count, s_words);
    fetch_chunk(gr, j, count, s_words + kChunk * kRoundThreads);
    fetch_chunk(vr, j, count, s_words + 2 * kChunk * kRoundThreads);
    // Some row of the block where the lane has no token.
    const float *p = kept + static_cast<int64_t>(min(at.group + j / kChunk, last_chunk)) * c.width;
#pragma unroll
    for (int v = 0; v < V; ++v)
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void *)(p + v),
          (__attribute__((address_space(3))) void *)(s_words + (3 * kChunk + v) * kRoundThreads +
                                                     wave_index() * 64),
          4, 0, 0);
  };
  int32_t j = (total - 1) / span * span;
  fetch(j);
  int turn = 0;
  for (; j >= 0; j -= span, turn ^= 1) {
    const int32_t t = at.lo + j;
    typename R::Word x[kChunk], g[kChunk], d[kChunk];
    float h[V];
    words_arrived();
    take_chunk(s_words, x);
    take_chunk(s_words + kChunk * kRoundThreads, g);
    take_chunk(s_words + 2 * kChunk * kRoundThreads, d);
#pragma unroll
    for (int v = 0; v < V; ++v)
      h[v] = __uint_as_float(s_words[(3 * kChunk + v) * kRoundThreads + threadIdx.x]);
    if (j >= span) {
      words_taken();
      fetch(j - span);
    }
    // prior: the state before a token, less its x.
    float a[kChunk][V], b[kChunk][V], prior[kChunk][V], p[V], u[V], f[V];
#pragma unroll
    for (int k = 0; k < kChunk; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) gate_pair(R::value(g[k], v), a[k][v], b[k][v]);
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] = 1.0f, u[v] = 0.0f;
    const bool plain = plain_backward(q, t, at.hi);
    bool fine = plain;
    if (plain) {
      float h1[V];
      Least least[V];
#pragma unroll
      for (int v = 0; v < V; ++v) h1[v] = h[v];
#pragma unroll
      for (int k = 0; k < kChunk; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float xv = R::value(x[k], v);
          prior[k][v] = h1[v] - xv;
          h1[v] = fmaf(a[k][v], h1[v], b[k][v] * xv);
        }
#pragma unroll
      for (int k = kChunk - 1; k >= 0; --k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          u[v] = a[k][v] * (R::value(d[k], v) + u[v]);
          p[v] *= a[k][v];
          least[v].add(a[k][v]);
        }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        fine = fine && finite(u[v]) && finite(p[v]) && finite(h1[v]);
        p[v] = least[v].marked(p[v]);
      }
      fine = __all(fine);
    }
    if (!fine) {
#pragma unroll
      for (int v = 0; v < V; ++v) p[v] = 1.0f, u[v] = 0.0f;
      Cursor w = q;
      if (j < count && t < w.first) w.previous(c, t);
#pragma unroll
      for (int k = 0; k < kChunk; ++k) {
        if (j + k < count) {
          if (t + k > w.last) w.next(c, t + k);
          if (t + k == w.first) load_state<V>(initial, c, at, w.s, h);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float xv = R::value(x[k], v);
            prior[k][v] = h[v] - xv;
            h[v] = applied<true>(a[k][v], h[v], scaled<true>(b[k][v], xv));
          }
        }
      }
      w = q;
#pragma unroll
      for (int k = kChunk - 1; k >= 0; --k) {
        if (j + k < count) {
          if (t + k < w.first) w.previous(c, t + k);
          const bool last = t + k == w.last;
          float f0[V];
          if (last) load_state<V>(v_final, c, at, w.s, f0);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            u[v] = scaled<true>(a[k][v], R::value(d[k], v) + (last ? f0[v] : u[v]));
            p[v] = last || a[k][v] == 0.0f ? -1.0f : p[v] * a[k][v];
          }
        }
      }
#pragma unroll
      for (int v = 0; v < V; ++v) p[v] = in_range(p[v]);
    }
    enter_chunk<V, true>(s_rounds, turn, c, at, p, u, carry, f);
    if (fine) {
      float f1[V];
#pragma unroll
      for (int v = 0; v < V; ++v) f1[v] = f[v];
#pragma unroll
      for (int k = kChunk - 1; k >= 0; --k) {
        Pack<T, V> dx, dg;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float gk = R::value(d[k], v) + f1[v], vx = b[k][v] * gk;
          f1[v] = a[k][v] * gk;
          dx.v[v] = static_cast<T>(vx);
          dg.v[v] = static_cast<T>(a[k][v] * (vx * prior[k][v]));
        }
        if (at.inside) {
          dxr.store(j + k, __builtin_bit_cast(typename R::Word, dx));
          dgr.store(j + k, __builtin_bit_cast(typename R::Word, dg));
        }
      }
#pragma unroll
      for (int v = 0; v < V; ++v) fine = fine && finite(f1[v]);
      if (__all(fine)) continue;
    }
#pragma unroll
    for (int k = kChunk - 1; k >= 0; --k) {
      if (j + k < count) {
        if (t + k < q.first) q.previous(c, t + k);
        if (t + k == q.last) load_state<V>(v_final, c, at, q.s, f);
        Pack<T, V> dx, dg;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float gk = R::value(d[k], v) + f[v], vx = scaled<true>(b[k][v], gk);
          const float vg = a[k][v] * (vx * prior[k][v]);
          dx.v[v] = static_cast<T>(vx);
          dg.v[v] = static_cast<T>(a[k][v] == 0.0f || b[k][v] == 0.0f ? 0.0f : vg);
          f[v] = scaled<true>(a[k][v], gk);
        }
        if (at.inside) {
          dxr.store(j + k, __builtin_bit_cast(typename R::Word, dx));
          dgr.store(j + k, __builtin_bit_cast(typename R::Word, dg));
          if (t + k == q.first && v_initial != nullptr) {
#pragma unroll
            for (int v = 0; v < V; ++v)
              v_initial[c.state_row(q.s) * c.width + at.col + v] = f[v];
          }
        }
      }
    }
  }
}

__global__ __launch_bounds__(kThreads) void scan_empty_kernel(Tokens c,
                                                              const float *__restrict__ in,
                                                              float *__restrict__ out) {
  empty_state(c, static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, in, out);
}

// One token per sequence, the decode form: nothing to scan.  64 x 128 bf16: 2.8
// us, the launch.
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
    float a, b;
    gate_pair(static_cast<float>(gs.v[v]), a, b);
    const float h = applied<true>(a, h0, scaled<true>(b, static_cast<float>(xs.v[v])));
    out.v[v] = static_cast<T>(h);
    final[t * width + col + v] = h;
  }
  store_pack<T, V>(y + t * width + col, out);
}

// ---------------------------------------------------------------- host ---

// The threads that a packed call spreads the tokens over, in waves per CU.  A
// lane of 16-bit rows holds two channels, so half the waves have as much in
// flight: 500k x 64 bf16 74.6 us with 16 and 82.8 us with 32, 200k x 99 f32
// (forward and backward) 328 and 315 us (270 now).
constexpr int64_t kSpread16 = 256 * 16 * 64, kSpread32 = 256 * 32 * 64;

struct Plan {
  Mode mode;
  int V;
  uint32_t slices;
  int64_t blocks;
  int threads;
  Tokens c;
  int64_t groups() const { return threads >> c.lane_bits; }
  int64_t strips() const { return blocks * groups(); }
  int64_t kept_rows() const {
    return mode == kRounds ? blocks * ceil_div(c.block, kChunk) : strips() * (c.steps / kChunk);
  }
};

// The plan depends on sizes and types alone, so a backward call finds its
// forward's.
Plan plan_of(int type, const int32_t *offsets, int64_t n, int64_t sequences, int64_t length,
             int64_t width, bool ragged, int32_t reverse) {
  Plan p{};
  Tokens &c = p.c;
  c.offsets = offsets;
  c.n = n;
  c.length = length;
  c.sequences = static_cast<int32_t>(sequences);
  c.reverse = reverse != 0;
  c.width = static_cast<uint32_t>(width);
  // 4 bytes per lane where 16-bit rows allow; 64 bytes of a row per block.
  p.V = type != R2S_TYPE_F32 && width % 2 == 0 ? 2 : 1;
  const int64_t vpr = width / p.V;
  auto set_lanes = [&](uint32_t most) {
    c.lane_bits = 0;
    while (c.lane_bits < most && (1 << c.lane_bits) < vpr) ++c.lane_bits;
    p.slices = static_cast<uint32_t>(ceil_div(vpr, 1 << c.lane_bits));
  };
  set_lanes(4);
  const int64_t lanes = int64_t{1} << c.lane_bits;
  if (!ragged && length <= 128) {
    // As many bytes of a row as leave no more lanes idle than 64 bytes do:
    // 500 x 100 x 512 f32, forward and back, 185 us with 256 bytes, 204 with 128,
    // 257 with 64; 3000 x 100 x 64 f32 forward 54, 55 and 61.
    p.mode = kOwn;
    for (uint32_t bits = 6; bits > 4; --bits)
      if (align_up(vpr, int64_t{1} << bits) <= align_up(vpr, 16)) {
        set_lanes(bits);
        break;
      }
    p.threads = kThreads;
    c.strip = static_cast<int32_t>(length);
    c.block = p.groups() * length;
  } else if ((!ragged && sequences * p.slices >= 192) || (!ragged && n * lanes <= 32768)) {
    // Against the packed form, forward and back: 8 x 4096 x 1024 bf16 161 and
    // 185 us, 64 x 512 x 128 bf16 39 and 54, 200 x 1000 x 128 f32 199 and 278;
    // 6 x 2000 x 1024 bf16, 192 blocks, 82 and 84.  128 bytes of a row and not
    // 64 where that leaves a block for each CU: 8 x 4096 x 1024 f32 238 and 327
    // us, 1000 x 200 x 128 bf16 134 and 173; with 128 blocks (8 x 4096 x 1024
    // bf16) 262 and 161.
    p.mode = kRounds;
    const bool whole = sequences * p.slices < 192;
    c.block = whole ? n : length;
    if (!whole && sequences * ceil_div(vpr, 32) >= 256) set_lanes(5);
    // Ragged sequences are packed however few there are: 893 tokens of 51, 256
    // channels, f32, 46 us forward and back, and 138 in rounds of one block.
    // At least two rounds, for the overlap: 1000 x 200 x 128 bf16 took 192 us
    // with one of 512 threads and 146 with two of 256; 1024 threads where they
    // fit, 179 us against 134 for 32 x 1024 x 1024 bf16.
    p.threads = 64;
    while (p.threads < kRoundThreads && p.groups() * 2 * kChunk < c.block) p.threads *= 2;
    c.strip = kChunk;
  } else {
    p.mode = kPacked;
    p.threads = kThreads;
    // 256 bytes of a row where that leaves no more lanes idle than 128: 200k x 99
    // f32, forward and back, 268 and 310 us, 30k x 1024 bf16 of 30 sequences 179
    // and 208; 200k x 70 f32, 128 lanes for 96, 211 and 188.
    set_lanes(align_up(vpr, 64) <= align_up(vpr, 32) ? 6 : 5);
    const int64_t even = ceil_div(n * (int64_t{p.slices} << c.lane_bits),
                                  p.V == 2 ? kSpread16 : kSpread32);
    c.strip = static_cast<int32_t>(
        align_up(std::min<int64_t>(std::max<int64_t>(even, 16), 128), kChunk));
    c.block = p.groups() * c.strip;
  }
  c.steps = static_cast<int32_t>(align_up(c.strip, kChunk));
  p.blocks = ceil_div(n, c.block);
  return p;
}

struct ScanSpace {
  float *strips, *blocks, *carries;
};
ScanSpace carve_scan(Carver &cv, const Plan &p) {
  ScanSpace s{};
  if (p.mode != kPacked) return s;
  s.strips = cv.take<float>(p.strips() * 2 * p.c.width);
  s.blocks = cv.take<float>(p.blocks * 2 * p.c.width);
  s.carries = cv.take<float>(p.blocks * p.c.width);
  return s;
}

int check_scan(const char *what, int type, const int32_t *offsets, int64_t n, int64_t sequences,
               int64_t length, int64_t width, std::initializer_list<int64_t> strides) {
  R2S_REQUIRE(known_type(type), "%s: unknown element type %d", what, type);
  R2S_REQUIRE(n >= 0 && sequences >= 0 && length >= 0 && width >= 0, "%s: negative size", what);
  R2S_REQUIRE(offsets != nullptr || n == sequences * length,
              "%s: %lld tokens are not %lld sequences of %lld", what, (long long)n,
              (long long)sequences, (long long)length);
  R2S_REQUIRE(sequences > 0 || n == 0, "%s: tokens without a sequence", what);
  // Token numbers are 32 bits wide, with room for a strip past the last.
  if (n > kInt32Max - (1 << 24) || sequences >= kInt32Max || width > (1 << 16)) {
    set_error("%s: more than 2^31 - 2^24 tokens, 2^31 - 1 sequences or 2^16 channels", what);
    return R2S_ERANGE;
  }
  for (int64_t s : strides) R2S_REQUIRE(s >= width, "%s: rows overlap", what);
  return R2S_OK;
}

// The limits of a plan: grid sizes, and the 32-bit lane offsets of Rows.
int check_plan(const char *what, int type, const Plan &p, std::initializer_list<int64_t> strides) {
  bool fits = p.blocks * p.slices <= kInt32Max && p.c.strip < (1 << 23);
  for (int64_t s : strides)
    fits &= s * type_size(type) * p.c.strip * (64 >> p.c.lane_bits) <= 0xffffffffll;
  if (!fits) {
    set_error("%s: rows too far apart or too many tokens", what);
    return R2S_ERANGE;
  }
  return R2S_OK;
}

int64_t states(const Tokens &c) { return static_cast<int64_t>(c.sequences) * c.width; }

// A launch for the sequences without a token, where there can be any.
int empty_states(const Tokens &c, const float *in, float *out, hipStream_t stream) {
  const int64_t blocks = ceil_div(states(c), kThreads);
  if (out == nullptr || blocks == 0 || (c.offsets == nullptr && c.length > 0)) return R2S_OK;
  scan_empty_kernel<<<dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, stream>>>(c, in,
                                                                                         out);
  return check_launch("gated_scan empty sequences");
}

// The maps of a packed call's strips and blocks, and the states that enter
// the blocks; empty_out [sequences][width] receives empty_in for the sequences
// without a token.
template <typename T, int V, bool kBack>
int packed_maps(const Plan &p, const T *a, int64_t as, const T *b, int64_t bs, const float *state,
                const float *empty_in, float *empty_out, const ScanSpace &s, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(p.blocks * p.slices));
  scan_maps_kernel<T, V, kBack><<<grid, dim3(kThreads), kThreads * V * 2 * sizeof(float),
                                  stream>>>(a, as, b, bs, state, p.c, p.slices, s.strips,
                                            s.blocks);
  R2S_RETURN_IF(check_launch("gated_scan maps"));
  const int64_t channel_blocks = ceil_div(p.c.width, kCarryCols);
  const int64_t empty_blocks =
      p.c.offsets != nullptr && empty_out != nullptr ? ceil_div(states(p.c), 1024) : 0;
  scan_carry_kernel<<<dim3(static_cast<uint32_t>(channel_blocks + empty_blocks)), dim3(1024), 0,
                      stream>>>(reinterpret_cast<const float2 *>(s.blocks),
                                static_cast<int32_t>(p.blocks), p.c, kBack ? 1 : 0,
                                static_cast<uint32_t>(channel_blocks), s.carries, empty_in,
                                empty_out);
  return check_launch("gated_scan carries");
}

template <typename T, int V>
int scan_fwd(const Plan &p, const void *x, int64_t xs, const void *g, int64_t gs,
             const float *initial, void *y_, float *final, float *kept, const ScanSpace &s,
             hipStream_t stream) {
  const Tokens &c = p.c;
  const T *xt = static_cast<const T *>(x), *gt = static_cast<const T *>(g);
  T *y = static_cast<T *>(y_);
  if (c.offsets == nullptr && c.length == 1) {
    const int64_t blocks = ceil_div(c.n * (c.width / V), kThreads);
    if (blocks > kInt32Max) {
      set_error("gated_scan_fwd: too many tokens");
      return R2S_ERANGE;
    }
    scan_step_kernel<T, V><<<dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, stream>>>(
        xt, xs, gt, gs, initial, c.n, c.width, y, final);
    return check_launch("gated_scan_fwd");
  }
  const dim3 grid(static_cast<uint32_t>(p.blocks * p.slices)), block(p.threads);
  if (p.mode == kPacked) {
    R2S_RETURN_IF((packed_maps<T, V, false>(p, xt, xs, gt, gs, initial, initial, final, s, stream)));
    scan_fwd_kernel<T, V, kPacked><<<grid, block, 0, stream>>>(
        xt, xs, gt, gs, initial, c, p.slices, s.strips, s.carries, kept, y, final);
  } else if (p.mode == kOwn) {
    scan_fwd_kernel<T, V, kOwn><<<grid, block, 0, stream>>>(
        xt, xs, gt, gs, initial, c, p.slices, nullptr, nullptr, kept, y, final);
  } else {
    scan_fwd_rounds_kernel<T, V><<<grid, block, 0, stream>>>(xt, xs, gt, gs, initial, c, p.slices,
                                                             kept, y, final);
  }
  return check_launch("gated_scan_fwd");
}

template <typename T, int V>
int scan_bwd(const Plan &p, const void *x, int64_t xs, const void *g, int64_t gs,
             const float *initial, const float *kept, const void *v_y, int64_t vs,
             const float *v_final, void *v_x, void *v_gate, float *v_initial, const ScanSpace &s,
             hipStream_t stream) {
  const Tokens &c = p.c;
  const T *xt = static_cast<const T *>(x), *gt = static_cast<const T *>(g);
  const T *vt = static_cast<const T *>(v_y);
  T *dx = static_cast<T *>(v_x), *dg = static_cast<T *>(v_gate);
  const dim3 grid(static_cast<uint32_t>(p.blocks * p.slices)), block(p.threads);
  if (p.mode == kPacked) {
    R2S_RETURN_IF((packed_maps<T, V, true>(p, gt, gs, vt, vs, v_final, v_final, v_initial, s, stream)));
    scan_bwd_kernel<T, V, kPacked><<<grid, block, 0, stream>>>(
        xt, xs, gt, gs, initial, vt, vs, v_final, c, p.slices, s.strips, s.carries, kept, dx, dg,
        v_initial);
  } else if (p.mode == kOwn) {
    scan_bwd_kernel<T, V, kOwn><<<grid, block, 0, stream>>>(
        xt, xs, gt, gs, initial, vt, vs, v_final, c, p.slices, nullptr, nullptr, kept, dx, dg,
        v_initial);
  } else {
    scan_bwd_rounds_kernel<T, V><<<grid, block, 0, stream>>>(
        xt, xs, gt, gs, initial, vt, vs, v_final, c, p.slices, kept, dx, dg, v_initial);
  }
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

int64_t r2s_gated_scan_kept_rows(int32_t type, int32_t ragged, int64_t sequences, int64_t length,
                                 int64_t n, int64_t width) {
  if (!r2s::known_type(type) || n <= 0 || width <= 0) return 0;
  return r2s::plan_of(type, nullptr, n, sequences, length, width, ragged != 0, 0).kept_rows();
}

int64_t r2s_gated_scan_workspace_bytes(int32_t type, int32_t ragged, int64_t sequences,
                                       int64_t length, int64_t n, int64_t width) {
  if (!r2s::known_type(type) || n <= 0 || width <= 0) return 0;
  r2s::Carver cv(nullptr);
  r2s::carve_scan(cv, r2s::plan_of(type, nullptr, n, sequences, length, width, ragged != 0, 0));
  return static_cast<int64_t>(cv.used);
}

int r2s_gated_scan_fwd(const void *x, int64_t x_stride, const void *gate, int64_t gate_stride,
                       const float *initial, const int32_t *offsets, int64_t sequences,
                       int64_t length, int64_t n, int64_t width, int32_t type, int32_t reverse,
                       void *y, float *final_state, float *kept, void *ws, size_t ws_bytes,
                       r2s_stream_t st) {
  using namespace r2s;
  clear_error();
  R2S_RETURN_IF(check_scan("gated_scan_fwd", type, offsets, n, sequences, length, width,
                           {x_stride, gate_stride}));
  if (width == 0 || sequences == 0) return R2S_OK;
  R2S_REQUIRE(final_state != nullptr, "gated_scan_fwd: null final states");
  const bool ragged = offsets != nullptr;
  hipStream_t stream = as_stream(st);
  Tokens all{};
  all.offsets = offsets;
  all.length = length;
  all.sequences = static_cast<int32_t>(sequences);
  all.width = static_cast<uint32_t>(width);
  if (n == 0) return empty_states(all, initial, final_state, stream);
  const Plan p = plan_of(type, offsets, n, sequences, length, width, ragged, reverse);
  R2S_RETURN_IF(check_plan("gated_scan_fwd", type, p, {x_stride, gate_stride, width}));
  R2S_REQUIRE(x != nullptr && gate != nullptr && y != nullptr,
              "gated_scan_fwd: null tokens or output");
  const int64_t need =
      r2s_gated_scan_workspace_bytes(type, ragged, sequences, length, n, width);
  if (need > 0 && (ws == nullptr || static_cast<int64_t>(ws_bytes) < need)) {
    set_error("gated_scan_fwd: workspace of %zu bytes, %lld required", ws_bytes, (long long)need);
    return R2S_EWORKSPACE;
  }
  Carver cv(ws);
  const ScanSpace s = carve_scan(cv, p);
  R2S_REQUIRE(p.V == 1 || pairs_fit({x, gate, y}, {x_stride, gate_stride}),
              "gated_scan_fwd: rows of 16-bit elements must start at multiples of 4 bytes");
  if (p.mode != kPacked) R2S_RETURN_IF(empty_states(p.c, initial, final_state, stream));
  R2S_BY_TYPE(type, {
    if constexpr (sizeof(T) == 2) {
      if (p.V == 2)
        return scan_fwd<T, 2>(p, x, x_stride, gate, gate_stride, initial, y, final_state, kept, s,
                              stream);
    }
    return scan_fwd<T, 1>(p, x, x_stride, gate, gate_stride, initial, y, final_state, kept, s,
                          stream);
  });
  return R2S_OK;
}

int r2s_gated_scan_bwd(const void *x, int64_t x_stride, const void *gate, int64_t gate_stride,
                       const float *initial, const int32_t *offsets, const float *kept,
                       const void *v_y, int64_t v_y_stride, const float *v_final,
                       int64_t sequences, int64_t length, int64_t n, int64_t width, int32_t type,
                       int32_t reverse, void *v_x, void *v_gate, float *v_initial, void *ws,
                       size_t ws_bytes, r2s_stream_t st) {
  using namespace r2s;
  clear_error();
  R2S_RETURN_IF(check_scan("gated_scan_bwd", type, offsets, n, sequences, length, width,
                           {x_stride, gate_stride, v_y_stride}));
  if (width == 0 || sequences == 0) return R2S_OK;
  const bool ragged = offsets != nullptr;
  hipStream_t stream = as_stream(st);
  Tokens all{};
  all.offsets = offsets;
  all.length = length;
  all.sequences = static_cast<int32_t>(sequences);
  all.width = static_cast<uint32_t>(width);
  if (n == 0) return empty_states(all, v_final, v_initial, stream);
  const Plan p = plan_of(type, offsets, n, sequences, length, width, ragged, reverse);
  R2S_RETURN_IF(check_plan("gated_scan_bwd", type, p,
                           {x_stride, gate_stride, v_y_stride, width}));
  R2S_REQUIRE(x != nullptr && gate != nullptr && v_y != nullptr && kept != nullptr &&
                  v_x != nullptr && v_gate != nullptr,
              "gated_scan_bwd: null tokens, gradients or kept states");
  const int64_t need =
      r2s_gated_scan_workspace_bytes(type, ragged, sequences, length, n, width);
  if (need > 0 && (ws == nullptr || static_cast<int64_t>(ws_bytes) < need)) {
    set_error("gated_scan_bwd: workspace of %zu bytes, %lld required", ws_bytes, (long long)need);
    return R2S_EWORKSPACE;
  }
  Carver cv(ws);
  const ScanSpace s = carve_scan(cv, p);
  R2S_REQUIRE(p.V == 1 || pairs_fit({x, gate, v_y, v_x, v_gate},
                                    {x_stride, gate_stride, v_y_stride}),
              "gated_scan_bwd: rows of 16-bit elements must start at multiples of 4 bytes");
  if (p.mode != kPacked) R2S_RETURN_IF(empty_states(p.c, v_final, v_initial, stream));
  R2S_BY_TYPE(type, {
    if constexpr (sizeof(T) == 2) {
      if (p.V == 2)
        return scan_bwd<T, 2>(p, x, x_stride, gate, gate_stride, initial, kept, v_y, v_y_stride,
                              v_final, v_x, v_gate, v_initial, s, stream);
    }
    return scan_bwd<T, 1>(p, x, x_stride, gate, gate_stride, initial, kept, v_y, v_y_stride,
                          v_final, v_x, v_gate, v_initial, s, stream);
  });
  return R2S_OK;
}

}  // extern "C"
