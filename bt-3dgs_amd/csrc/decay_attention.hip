// Linear attention with a decay for each head, over sequences of tokens:
//
//   S_t = g S_{t-1} + k_t v_t^T,   y_t = s S_t^T q_t,   g = exp(log_decay).
//
// A sequence is walked in chunks of C tokens.  With i, j the tokens of a chunk and S
// the state before it,
//
//   y_i = s (g^(i+1) S^T q_i + sum_{j <= i} g^(i-j) (q_i k_j) v_j),
//   S' = g^C S + sum_j g^(C-1-j) k_j v_j^T,
//
// four products on the matrix cores.  No power is negative: the weights g^(i-j) are
// made for the pairs, so a strong decay underflows to the zeros it means.
//
// The backward is the same walk three times, of other inputs:
//
//   dq: S (as its transpose) from dy, v, k in the forward's order,
//   dv: R_t = g R_{t+1} + s q_t dy_t^T from k, q, dy from the other end,
//   dk: R (as its transpose) from v, dy, q from the other end,
//
// where R begins with the last state's gradient before any decay: "early" roles
// decay a state behind its token, g^i and g^(C-j) above.  g R after the last token is
// the first state's gradient.
//
// A block is one head and up to 16 W columns of v of one span of a sequence (of heads
// up to 16 channels, four heads of a wave each).  Each of a head's W waves keeps the
// state's rows of 16 columns in registers and brings them up to date; the outputs are
// shared out by tokens instead, so that each score is made once for up to 64 columns,
// and every wave reads the state of all the block's columns, as operands, from LDS.
// The products are made transposed (scores as k q^T, outputs as v^T p): then an
// accumulator's values are, lane by lane, the next product's operand, and a lane
// ends with neighbouring columns of one token.
//
// Precision: the scores, the state and the decayed v are float32 values.  As
// operands of 16-bit products they are split into bfloat16 parts, each the rounding of
// what the parts before leave, with a product for each.  The decayed v, which adds up
// in the float32 state, has three, which hold its 24 bits.  Scores and state, whose
// products end in a 16-bit output, have two: these leave out at most 2^-17 of a value,
// where the output's own rounding is 2^-8 (bfloat16) or 2^-11 (float16).  Three there
// take 335 us where two take 303 (8 x 4096 x 16 x 64 bfloat16, both ways) and 127
// where 118 (500k x 4 x 16, forward).  float16 inputs beside them, whose range does not
// hold those values, are split without loss into two bfloat16 parts, at a product more
// for each: 446 us both ways of the former where bfloat16 takes 299, and 123 forward of
// the latter where 98.
//
// A zero weight times a NaN or an infinity is a NaN: a chunk with such a v would
// reach back to its earlier tokens.  Its tokens are walked one by one.
//
// Few sequences are cut into spans: their own states first (k and v alone), one
// pass along each sequence over those, and then all spans at once from the states
// before them.
#include <algorithm>

#include "r2s_latent.h"

namespace r2s {
namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using i16x4 = __attribute__((ext_vector_type(4))) short;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

constexpr int kMostChannels = 256;
constexpr int64_t kMostStep = 1 << 24;  // elements between tokens: a chunk is within 2^31 bytes

// One input: sequence s (of equal ones), its token and head by strides.
struct View {
  const void *p;
  int64_t sequence, token, head;
};

// One walk: the names are those of the forward's.
struct Role {
  View q, k, v;
  const float *initial;  // [sequences][heads][state], may be null: zeros
  float *carried;        // [cuts][heads][state]: the state behind each span but the last
  int32_t dk, dv;
  int32_t transposed;    // initial and carried are stored [dv][dk]
  int32_t early, backwards;
  float scale_in, scale_out;  // of k v^T, and of everything that is read
  void *y;                    // [n][heads][dv]
  float *final_state;         // [sequences][heads][dk][dv], may be null
};

constexpr int kRoles = 3;

// How the sequences are cut.
struct Cut {
  const int32_t *offsets;  // ragged
  const int32_t *order;    // ragged, several spans: items as they are taken, see below
  const int32_t *index;    // [wholes], the span of the first of them, -1: the last
  const int32_t *first;    // and each sequence's first item, as places are counted
  int64_t n, sequences, length, span;
  int64_t carried;  // places for states between spans
  int32_t spans;    // of an equal sequence
  int32_t wholes;   // spans that ragged sequences may fill at most
};

struct Walk {
  Role role[kRoles];
  const float *log_decay;
  Cut cut;
  int32_t heads, column_blocks;
  uint32_t roles;
  uint32_t blocks, together;  // and how many of them one XCD takes in a row; 0: its share
  uint32_t first;             // block of this launch
};

// A block's span of its sequence: tokens [at, at + count) of the walk's order.
struct Span {
  int64_t sequence, lo, length;  // the sequence's first token and tokens
  int64_t at, count;
  int64_t place;  // among the carried states
  bool first, last;
};

__device__ __forceinline__ int64_t bound(const Cut &c, int64_t s) {
  return min(max(static_cast<int64_t>(c.offsets[s]), int64_t{0}), c.n);
}

// False for an item that there is not.  Sequence `sequences` stands for the
// tokens behind the last one.
__device__ __forceinline__ bool find_span(const Cut &c, int64_t item, Span &x) {
  int64_t sequence = item, index = 0, items = 1, place = 0, lo = 0, length = c.length;
  if (c.offsets == nullptr) {
    const uint32_t which = static_cast<uint32_t>(item), spans = static_cast<uint32_t>(c.spans);
    sequence = which / spans;
    index = which % spans;
    items = c.spans;
    lo = sequence * length;
    place = sequence * (items - 1) + index;
  } else {
    if (c.order != nullptr) {
      sequence = c.order[item];
      if (sequence < 0) return false;
      index = item < c.wholes ? c.index[item] : -1;
      const int64_t first = c.first[sequence];
      items = c.first[sequence + 1] - first;
      if (index < 0) index = max(items - 1, int64_t{0});  // offsets may be anything
      place = first + index - sequence;  // each sequence before has an item without a place
    }
    lo = bound(c, sequence);
    const int64_t hi = sequence < c.sequences ? bound(c, sequence + 1) : c.n;
    length = max(hi - lo, int64_t{0});
  }
  x.sequence = sequence;
  x.lo = lo;
  x.length = length;
  x.place = place;
  x.at = index * c.span;
  x.count = max(min(length - x.at, c.span), int64_t{0});
  x.first = index == 0;
  x.last = index + 1 >= items;
  // Offsets that do not ascend may ask for more places than there are.
  return place >= 0 && (x.last || place < c.carried) &&
         (x.first || (place > 0 && place <= c.carried));
}

// The items of ragged sequences: every sequence's spans, at least one, those of the
// tokens behind the last, and -1 for places left over.  Whole spans come first, then
// each sequence's rest, the longest first in classes of an eighth of a span: with
// short ones last, the device runs dry all at once (100k tokens in 512 sequences, 3
// heads of 33 x 45 float32: forward 166 to 174 us, in the order of the sequences and in equal
// shares to the XCDs 231).
constexpr uint32_t kEighths = 8, kClasses = 1 + kEighths;
__global__ __launch_bounds__(1024) void decay_items_kernel(Cut c, int64_t most,
                                                           int32_t *__restrict__ order,
                                                           int32_t *__restrict__ index,
                                                           int32_t *__restrict__ first) {
  __shared__ int64_t s_total[16];
  __shared__ unsigned long long s_next[kClasses];  // offsets that do not ascend add up to much
  if (threadIdx.x < kClasses) s_next[threadIdx.x] = 0;
  __syncthreads();
  auto tokens_of = [&](int64_t s) {
    const int64_t hi = s < c.sequences ? bound(c, s + 1) : c.n;
    return max(hi - bound(c, s), int64_t{0});
  };
  // Of the tokens behind a sequence's whole spans, if there are any.
  auto class_of = [&](int64_t rest) {
    return kEighths - static_cast<uint32_t>((rest * kEighths - 1) / c.span);
  };
  int64_t before = 0;
  for (int64_t s0 = 0; s0 <= c.sequences; s0 += 1024) {
    const int64_t s = s0 + threadIdx.x;
    int64_t items = 0;
    if (s <= c.sequences) {
      const int64_t tokens = tokens_of(s), whole = tokens / c.span, rest = tokens - whole * c.span;
      items = whole + (rest > 0 ? 1 : 0);
      if (whole > 0) atomicAdd(&s_next[0], static_cast<unsigned long long>(whole));
      if (rest > 0) atomicAdd(&s_next[class_of(rest)], 1ull);
      if (s < c.sequences && items == 0) {
        items = 1;
        atomicAdd(&s_next[kClasses - 1], 1ull);
      }
    }
    const int64_t inside = wave_inclusive_scan(items);
    if (lane_id() == 63) s_total[wave_index()] = inside;
    __syncthreads();
    int64_t at = before + inside - items;
    for (uint32_t w = 0; w < 16; ++w) {
      if (w < wave_index()) at += s_total[w];
      before += s_total[w];
    }
    // Offsets that do not ascend may name more items than there is room for.
    before = min(before, most);
    if (s <= c.sequences) first[s] = static_cast<int32_t>(min(at, most));
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    first[c.sequences + 1] = static_cast<int32_t>(before);
    unsigned long long sum = 0;
    for (uint32_t i = 0; i < kClasses; ++i) {
      const unsigned long long own = s_next[i];
      s_next[i] = sum;
      sum += own;
    }
  }
  __syncthreads();
  auto put = [&](int64_t at, int64_t s, int64_t span) {
    if (at < most) order[at] = static_cast<int32_t>(s);
    if (at < min(most, static_cast<int64_t>(c.wholes))) index[at] = static_cast<int32_t>(span);
  };
  for (int64_t s0 = 0; s0 <= c.sequences; s0 += 1024) {
    const int64_t s = s0 + threadIdx.x;
    int64_t whole = 0, at = 0;
    if (s <= c.sequences) {
      const int64_t tokens = tokens_of(s), rest = tokens - tokens / c.span * c.span;
      whole = tokens / c.span;
      if (whole > 0) at = atomicAdd(&s_next[0], static_cast<unsigned long long>(whole));
      if (rest > 0) put(atomicAdd(&s_next[class_of(rest)], 1ull), s, -1);
      if (s < c.sequences && tokens == 0) put(atomicAdd(&s_next[kClasses - 1], 1ull), s, -1);
    }
    for (uint64_t some = ballot(whole > 0); some != 0; some &= some - 1) {
      const uint32_t from = static_cast<uint32_t>(__builtin_ctzll(some));
      const int64_t spans = readlane_i64(whole, from), to = readlane_i64(at, from);
      for (int64_t i = lane_id(); i < spans; i += 64) put(to + i, s - lane_id() + from, i);
    }
  }
  for (int64_t i = before + threadIdx.x; i < most; i += 1024) order[i] = -1;
}

// The states behind `count` spans of a sequence from each span's own, from `now` on:
// p [count] of one element, `step` apart.  Returns the last; stores them with kStore.
template <bool kStore>
__device__ __forceinline__ float carry_along(float *p, int64_t step, int64_t count, float keep,
                                             float now) {
  constexpr int kAhead = 8;
  for (int64_t c = 0; c < count; c += kAhead) {
    float own[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) own[a] = c + a < count ? p[(c + a) * step] : 0.0f;
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (c + a < count) {
        now = fmaf(keep, now, own[a]);
        if constexpr (kStore) p[(c + a) * step] = now;
      }
    }
  }
  return now;
}

// Equal sequences of few spans: a thread to an element of their states.
__global__ __launch_bounds__(256) void decay_carry_few_kernel(Walk w, int64_t total) {
  const Role &r = w.role[0];
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const int64_t size = static_cast<int64_t>(r.dk) * r.dv, step = w.heads * size;
  const int64_t sequence = i / step, e = i - sequence * step, count = w.cut.spans - 1;
  const float keep = expf(w.log_decay[e / size] * static_cast<float>(w.cut.span));
  carry_along<true>(r.carried + sequence * count * step + e, step, count, keep,
                    r.initial != nullptr ? r.initial[i] : 0.0f);
}

// Any sequences: a block takes 64 elements of the states of `per` sequences, of which
// it looks at all together, as ragged ones mostly have one span.  Its 16 waves take
// a sequence of few spans each; of many they take a run of spans each, add it up, and
// go over it again from what the waves before them leave, so that hundreds of spans
// are not a chain of as many loads (four heads of 16 x 16: 600 spans in 11 us; a
// chain took 12 for 252).
__global__ __launch_bounds__(1024) void decay_carry_kernel(Walk w, int per) {
  __shared__ float s_sum[16][64];
  const Role &r = w.role[0];
  const int64_t size = static_cast<int64_t>(r.dk) * r.dv, step = w.heads * size;
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 64 + lane_id();
  const bool some = e < step;
  const uint32_t wave = wave_index();
  const float log_span = some ? w.log_decay[e / size] * static_cast<float>(w.cut.span) : 0.0f;
  const float keep = expf(log_span);
  auto begin = [&](int64_t sequence) {
    return r.initial != nullptr && some ? r.initial[sequence * step + e] : 0.0f;
  };
  for (int64_t s0 = static_cast<int64_t>(blockIdx.y) * per; s0 < w.cut.sequences;
       s0 += static_cast<int64_t>(gridDim.y) * per) {
    const int64_t mine = s0 + lane_id();
    int64_t place = 0, count = 0;
    if (static_cast<int>(lane_id()) < per && mine < w.cut.sequences) {
      place = mine * (w.cut.spans - 1);
      count = w.cut.spans - 1;
      if (w.cut.offsets != nullptr) {
        place = w.cut.first[mine] - mine;
        count = w.cut.first[mine + 1] - w.cut.first[mine] - 1;
        count = min(count, w.cut.carried - place);
      }
    }
    uint32_t turn = 0;
    for (uint64_t few = ballot(count > 0 && count <= 16); few != 0; few &= few - 1) {
      if (turn++ % 16 != wave) continue;
      const uint32_t from = static_cast<uint32_t>(__builtin_ctzll(few));
      carry_along<true>(r.carried + readlane_i64(place, from) * step + e, step,
                        some ? readlane_i64(count, from) : 0, keep, begin(s0 + from));
    }
    for (uint64_t many = ballot(count > 16); many != 0; many &= many - 1) {
      const uint32_t from = static_cast<uint32_t>(__builtin_ctzll(many));
      const int64_t spans = readlane_i64(count, from), each = (spans + 15) / 16;
      const int64_t lo = min(wave * each, spans), run = some ? min(each, spans - lo) : 0;
      float *p = r.carried + (readlane_i64(place, from) + lo) * step + e;
      s_sum[wave][lane_id()] = carry_along<false>(p, step, run, keep, 0.0f);
      __syncthreads();
      float now = begin(s0 + from);
      const float whole = expf(log_span * static_cast<float>(each));
      for (uint32_t i = 0; i < wave && run > 0; ++i) now = fmaf(whole, now, s_sum[i][lane_id()]);
      carry_along<true>(p, step, run, keep, now);
      __syncthreads();  // the sums have been read
    }
  }
}

// ------------------------------------------------------------ operands ---

template <typename T>
__device__ __forceinline__ f32x4 multiply(u32x4 a, u32x4 b, f32x4 acc) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], acc, 0, 0, 0);
    return acc;
  } else if constexpr (std::is_same<T, bf16_t>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
  }
}

// Float values of an operand's 16 bytes as a rounded part and the rounded rest, and
// with kThree what that leaves; float32 as they are.
template <typename T>
struct Parts {
  u32x4 high, rest, last;
};
template <typename T, bool kThree = false>
__device__ __forceinline__ Parts<T> split(const float (&x)[16 / sizeof(T)]) {
  Parts<T> out;
  if constexpr (sizeof(T) == 4) {
    out.high = __builtin_bit_cast(u32x4, f32x4{x[0], x[1], x[2], x[3]});
  } else {
    Pack<T, 8> high, rest, last;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      high.v[i] = static_cast<T>(x[i]);
      const float left = x[i] - static_cast<float>(high.v[i]);
      rest.v[i] = static_cast<T>(left);
      if constexpr (kThree) last.v[i] = static_cast<T>(left - static_cast<float>(rest.v[i]));
    }
    out.high = __builtin_bit_cast(u32x4, high);
    out.rest = __builtin_bit_cast(u32x4, rest);
    if constexpr (kThree) out.last = __builtin_bit_cast(u32x4, last);
  }
  return out;
}
template <typename T>
__device__ __forceinline__ void widen(u32x4 raw, float (&x)[16 / sizeof(T)]) {
  const Pack<T, 16 / sizeof(T)> p = __builtin_bit_cast(Pack<T, 16 / sizeof(T)>, raw);
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) x[i] = static_cast<float>(p.v[i]);
}

// The type that values are split in: float16's range does not hold scores and
// states, and the rests of decayed v's would be below its normal numbers.
template <typename T>
struct Wide {
  using type = T;
};
template <>
struct Wide<f16_t> {
  using type = bf16_t;
};

// An input beside them: float16's in two bfloat16 parts, which hold it exactly.
template <typename T>
__device__ __forceinline__ Parts<typename Wide<T>::type> beside(u32x4 raw) {
  if constexpr (std::is_same<T, f16_t>::value) {
    float x[8];
    widen<T>(raw, x);
    return split<bf16_t>(x);
  } else {
    return {raw, raw};
  }
}

// acc += a b of an input and split values, as rows and columns or the other way
// round.  T is the inputs' type; smaller products first.
template <typename T, bool kInputRows, bool kThree = false>
__device__ __forceinline__ f32x4 multiply_split(const Parts<typename Wide<T>::type> &input,
                                                const Parts<typename Wide<T>::type> &values,
                                                f32x4 acc) {
  using U = typename Wide<T>::type;
  auto go = [&](u32x4 a, u32x4 b) {
    acc = kInputRows ? multiply<U>(a, b, acc) : multiply<U>(b, a, acc);
  };
  if constexpr (sizeof(T) == 2) {
    if constexpr (kThree) go(input.high, values.last);
    if constexpr (kThree && std::is_same<T, f16_t>::value) go(input.rest, values.rest);
    if constexpr (std::is_same<T, f16_t>::value) go(input.rest, values.high);
    go(input.high, values.rest);
  }
  go(input.high, values.high);
  return acc;
}

// g^x for a whole number x of tokens; what is below float32's normal range is 0.
__device__ __forceinline__ float power(float log2_decay, int x) {
  return x == 0 ? 1.0f : __builtin_amdgcn_exp2f(log2_decay * static_cast<float>(x));
}

// --------------------------------------------------------------- walk ----

// Rows of D elements in LDS, 16 bytes apart from a power of two so that rows side by
// side start in different banks.
template <typename T, int D>
struct Tile {
  static constexpr int kPitch = D * static_cast<int>(sizeof(T)) + 16;
  static constexpr int kPer = 16 / static_cast<int>(sizeof(T));
};

// 16 bytes of the summed index along a row, from LDS.
template <typename T, int D>
__device__ __forceinline__ u32x4 along(const char *tile, int row, int piece) {
  return *reinterpret_cast<const u32x4 *>(tile + row * Tile<T, D>::kPitch + piece * 16);
}
// 16 bytes of the summed index across rows: 16 bits: rows 4 g to 4 g + 3 and 16
// on, g the lane's group of 16, of the lane's column; float32: rows 4 g to 4 g + 3.
// The lane's column is (i / 4) run + first + i % 4, i = lane % 16.
template <typename T, int D, int kRun>
__device__ __forceinline__ u32x4 across(const char *tile, int row, int first) {
  const int lane = static_cast<int>(lane_id()), i = lane % 16, g = lane / 16;
  if constexpr (sizeof(T) == 2) {
    // Sixteen lanes read 4 rows of 4 times 4 neighbours, 8 bytes each, and get 4
    // rows of one column each.
    const char *p = tile + (row + g * 4 + i / 4) * Tile<T, D>::kPitch +
                    (i % 4 * kRun + first) * 2;
    const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) i16x4 *)p);
    const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) i16x4 *)(p + 16 * Tile<T, D>::kPitch));
    u32x4 out;
    __builtin_memcpy(&out, &x, 8);
    __builtin_memcpy(reinterpret_cast<char *>(&out) + 8, &y, 8);
    return out;
  } else {
    const char *p = tile + (row + g * 4) * Tile<T, D>::kPitch + (i / 4 * kRun + first + i % 4) * 4;
    u32x4 out;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      out[j] = *reinterpret_cast<const uint32_t *>(p + j * Tile<T, D>::kPitch);
    return out;
  }
}

// A thread's number among the kThreads that share a head, and their meeting.  A head of
// one wave needs no barrier: a wave's LDS accesses are in order, and its heads
// beside it in the block go their own ways.
template <int kThreads>
__device__ __forceinline__ int head_thread() {
  return static_cast<int>(kThreads == 64 ? lane_id() : threadIdx.x);
}
template <int kThreads>
__device__ __forceinline__ void head_sync() {
  if constexpr (kThreads == 64) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  } else {
    __syncthreads();
  }
}

template <typename T, int V>
struct __attribute__((packed)) Loose {
  T v[V];
};

// The piece of 16 bytes of a row that holds its last `there` elements, where that is
// less than a piece: read as the row's last 16 bytes, and moved down.
template <typename T>
struct Tail {
  static constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  int back;  // elements that the read begins earlier
  __device__ __forceinline__ Tail(int there, int width)
      : back(there > 0 && there < kPer && width >= kPer ? kPer - there : 0) {}
  __device__ __forceinline__ u32x4 move(u32x4 x) const {
    constexpr int kWord = sizeof(T) == 4 ? 1 : 2;  // elements
#pragma unroll
    for (int step = kPer / 2; step > 0; step /= 2) {
      if (step >= kWord) {
        const int words = step / kWord;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t from = j + words < 4 ? x[j + words] : 0u;
          x[j] = (back & step) != 0 ? from : x[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t from = x[j] >> 16 | (j < 3 ? x[j + 1] << 16 : 0u);
          x[j] = (back & step) != 0 ? from : x[j];
        }
      }
    }
    return x;
  }
};
// A piece of a row: 16 bytes at `at` (Tail's place), of a row narrower than that
// element by element.
template <typename T, bool kWhole>
__device__ __forceinline__ u32x4 load_piece(const T *at, int there, const Tail<T> &tail) {
  constexpr int kPer = Tail<T>::kPer;
  if constexpr (kWhole) {
    return __builtin_bit_cast(u32x4, *reinterpret_cast<const Loose<T, kPer> *>(at));
  } else {
    if (there >= kPer || tail.back != 0)
      return tail.move(__builtin_bit_cast(u32x4, *reinterpret_cast<const Loose<T, kPer> *>(at)));
    Pack<T, kPer> e;
#pragma unroll
    for (int j = 0; j < kPer; ++j) e.v[j] = j < there ? at[j] : static_cast<T>(0.0f);
    return __builtin_bit_cast(u32x4, e);
  }
}

// A chunk's rows on their way to LDS: kCount pieces of 16 bytes a thread, of one
// column and rows kStep apart.  The addresses are a scalar one for each piece and an
// unsigned 32-bit offset of the thread's own, which is all that stays in vector
// registers.  kWhole: the width is a multiple of a piece.
template <typename T, int D, int C, int kThreads, bool kWhole>
struct Stage {
  static constexpr int kPieces = D * static_cast<int>(sizeof(T)) / 16;
  static constexpr int kStep = kThreads / kPieces;
  static constexpr int kCount = C / kStep;
  static constexpr int kPer = Tile<T, D>::kPer;
  static_assert(kThreads % kPieces == 0 && C % kStep == 0, "whole rows of pieces");
  u32x4 raw[kCount];
  uint32_t offset;
  int row, there;  // the first piece's row; elements of the width in the column's piece
  Tail<T> tail;
  // `step` elements between rows, at most 2^24 of either sign.
  __device__ __forceinline__ Stage(int64_t step, int width)
      : row(head_thread<kThreads>() / kPieces),
        there(width - head_thread<kThreads>() % kPieces * kPer), tail(there, width) {
    const int64_t rows = step >= 0 ? row * step : (kStep - 1 - row) * -step;
    offset = static_cast<uint32_t>(rows + (width - there) - (kWhole ? 0 : tail.back)) *
             static_cast<uint32_t>(sizeof(T));
  }
  // Rows from `first` on, `left` of them; zeros for those past them and for columns
  // past the width.
  __device__ __forceinline__ void load(const T *first, int64_t step, int64_t left) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const char *base = reinterpret_cast<const char *>(
          first + (i * kStep + (step < 0 ? kStep - 1 : 0)) * step);
      u32x4 x{0, 0, 0, 0};
      if (row + i * kStep < left && there > 0) {
        x = load_piece<T, kWhole>(reinterpret_cast<const T *>(base + offset), there, tail);
      }
      raw[i] = x;
    }
  }
  __device__ __forceinline__ void put(char *tile) const {
    char *p = tile + row * Tile<T, D>::kPitch + head_thread<kThreads>() % kPieces * 16;
#pragma unroll
    for (int i = 0; i < kCount; ++i)
      *reinterpret_cast<u32x4 *>(p + i * kStep * Tile<T, D>::kPitch) = raw[i];
  }
  // Whether an element is not finite.
  __device__ __forceinline__ bool bad() const {
    using u16x2 = __attribute__((ext_vector_type(2))) uint16_t;
    if constexpr (sizeof(T) == 4) {
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < kCount; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) most = max(most, raw[i][j] & 0x7FFFFFFFu);
      return most >= 0x7F800000u;
    } else {
      u16x2 most{0, 0};
#pragma unroll
      for (int i = 0; i < kCount; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          most = __builtin_elementwise_max(
              most, __builtin_bit_cast(u16x2, raw[i][j] & 0x7FFF7FFFu));
      const uint16_t least = std::is_same<T, bf16_t>::value ? 0x7F80 : 0x7C00;
      return most[0] >= least || most[1] >= least;
    }
  }
};

// A wave's rows of q as operands, straight from memory: tile `own` of 16 rows, row i
// and piece 4 kb + g of 16 bytes to a lane.
template <typename T, int KB, int kOwn, bool kWhole>
struct Rows {
  static constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  u32x4 raw[kOwn][KB];
  uint32_t offset;
  int row, width, channels;  // elements of a row from the lane's first on, and in all
  __device__ __forceinline__ Rows(int64_t step, int c) : channels(c) {
    row = static_cast<int>(lane_id()) % 16;
    const int column = static_cast<int>(lane_id()) / 16 * kPer;
    offset = static_cast<uint32_t>((step >= 0 ? row * step : (15 - row) * -step) + column) *
             static_cast<uint32_t>(sizeof(T));
    width = channels - column;
  }
  // The tiles first + own of `tiles` each; zeros past `left` rows and the width.
  __device__ __forceinline__ void load(const T *base, int64_t step, int64_t left, int first,
                                       int tiles) {
#pragma unroll
    for (int own = 0; own < kOwn; ++own) {
      const int it = first + own * tiles;
      const char *p = reinterpret_cast<const char *>(
          base + (it * 16 + (step < 0 ? 15 : 0)) * step);
      const bool some = it * 16 + row < left;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const T *at = reinterpret_cast<const T *>(p + offset) + kb * 4 * kPer;
        const int there = width - kb * 4 * kPer;
        const Tail<T> tail(kWhole ? 0 : there, channels);
        u32x4 x{0, 0, 0, 0};
        if (some && there > 0) x = load_piece<T, kWhole>(at - tail.back, there, tail);
        raw[own][kb] = x;
      }
    }
  }
};

// Zeros in the rows of a tile from the second on.
template <typename T, int D, int C, int kThreads>
__device__ __forceinline__ void clear_rows(char *tile) {
  constexpr int kPieces = D * static_cast<int>(sizeof(T)) / 16;
  for (int q = kPieces + head_thread<kThreads>(); q < C * kPieces; q += kThreads)
    *reinterpret_cast<u32x4 *>(tile + q / kPieces * Tile<T, D>::kPitch + q % kPieces * 16) =
        u32x4{0, 0, 0, 0};
}

// KD: channels of q and k that LDS and registers have room for; W waves.  kStates: the
// spans' own states, no outputs.
template <typename T, int KD, int W, bool kStates>
struct Shape {
  static constexpr int C = sizeof(T) == 4 || KD == 256 || W < 4 ? 32 : 64;  // tokens of a chunk
  static constexpr int kThreads = 64 * W, kColumns = 16 * W;
  static constexpr int kFragment = 64 / static_cast<int>(sizeof(T));  // summed by 16 bytes a lane
  static constexpr int kTiles = kFragment / 16;                       // tiles of 16 to a fragment
  static constexpr int KB = KD / kFragment, JB = C / kFragment;
  // Outputs: tiles of 16 tokens for each wave, or tokens by parts of the columns.
  static constexpr int IT = C / 16, kOwn = IT > W ? IT / W : 1, kPartsOfColumns = W > IT ? W / IT : 1;
  static constexpr int NT = W / kPartsOfColumns;  // column tiles of a wave's outputs
  static constexpr int kRun = 4 * NT;             // neighbouring columns of a lane's outputs
  static constexpr int kOperands = sizeof(T) == 4 ? 1 : 2;
  static constexpr int kK = C * Tile<T, KD>::kPitch, kV = C * Tile<T, kColumns>::kPitch;
  static constexpr int kS = kStates ? 0 : KB * W * kOperands * 1024;
  static constexpr int kLds = kK + kV + kS;
  // Heads of a block: four of one wave each, so that a compute unit reads the whole
  // lines that they share.
  static constexpr int kHeads = W == 1 ? 4 : 1;
  // Waves of a SIMD that the registers are shared out to.
  static constexpr int kPerSimd =
      KD == 32 ? (W == 1 && sizeof(T) == 4 ? 3 : 4) : KD == 64 ? 3 : KD == 128 ? 2 : 1;
};

// The walk.  8 sequences of 4096 tokens, 16 heads of 64 bfloat16: the spans' own
// states 29 to 34 us, the forward's walk 60 to 70 (3.8 to 4.5 TB/s of q, k, v and y), the
// backward's three roles 164 to 188.  What bounds it is not the memory: with all inputs in the cache the
// walk takes as long.  A wave issues some 330 vector, 65 LDS and 58 matrix
// instructions for a chunk, between two barriers that three blocks of a CU have to
// cover for each other; a fourth does not fit the registers (107 us for the whole
// forward, with spills, against 99).  500k tokens of 4 heads of 16: 26 and 60 us, where
// rows of 32 bytes and one wave to a head are the bound.  float32: the matrix cores,
// at 1/8 of the 16-bit rate, are busy half of the time; three bfloat16 products in
// place of a float32 one took 479 us at 8 x 4096 x 8 x 128, these 354 to 371.  Odd widths
// above 128 in float32 are past the registers (272 bytes of scratch a lane): 4 x 4096 x
// 4 x 131 takes 586 us forward, 132 channels 334.
template <typename T, int KD, int W, bool kStates, bool kWhole>
__global__ __launch_bounds__((64 * W * Shape<T, KD, W, kStates>::kHeads),
                             (Shape<T, KD, W, kStates>::kPerSimd)) void decay_walk_kernel(Walk w) {
  using S = Shape<T, KD, W, kStates>;
  constexpr int C = S::C, kThreads = S::kThreads, KB = S::KB, JB = S::JB, kTiles = S::kTiles;
  constexpr int kFragment = S::kFragment, kPer = Tile<T, KD>::kPer, NT = S::NT, kRun = S::kRun;
  constexpr int kRows = 4 * kTiles;  // neighbouring rows of the state in a lane
  using U = typename Wide<T>::type;
  extern __shared__ __attribute__((aligned(16))) char s_tile[];
  constexpr int kHeads = S::kHeads;
  __shared__ int s_bads[kHeads][2];
  __shared__ float s_lefts[kHeads][2 * C];
  const int inner = kHeads > 1 ? static_cast<int>(wave_index()) : 0;  // head of the block
  int *s_bad = s_bads[inner];
  float *s_left = s_lefts[inner];
  char *s_k = s_tile + inner * S::kLds, *s_v = s_k + S::kK, *s_s = s_v + S::kV;

  // Roles of the same tokens are neighbours, and neighbours share an XCD's cache.
  // Ragged items, long ones first, are dealt out to the XCDs in turn.
  uint32_t id = blockIdx.x;
  if (w.together == 0) {
    id = w.first + xcd_swizzle(id, gridDim.x);
  } else {
    id += w.first;
    const uint32_t turn = id / 8;
    id = (turn / w.together * 8 + id % 8) * w.together + turn % w.together;
    if (id >= w.blocks) return;
  }
  const Role &r = w.role[id % w.roles];
  id /= w.roles;
  const uint32_t head_blocks = static_cast<uint32_t>(w.heads + kHeads - 1) / kHeads;
  const uint32_t per_item = head_blocks * w.column_blocks;
  const uint32_t item = id / per_item, inside = id - item * per_item;
  const int head =
      static_cast<int>(inside / static_cast<uint32_t>(w.column_blocks)) * kHeads + inner;
  if (kHeads > 1 && head >= w.heads) return;
  const int block_column = static_cast<int>(inside % static_cast<uint32_t>(w.column_blocks)) *
                           S::kColumns;
  const int dk = r.dk, dv = r.dv;
  if (block_column >= dv) return;
  Span x;
  if (!find_span(w.cut, item, x)) return;
  x.sequence = uniform_value(x.sequence);
  x.lo = uniform_value(x.lo);
  x.length = uniform_value(x.length);
  x.at = uniform_value(x.at);
  x.count = uniform_value(x.count);
  x.place = uniform_value(x.place);
  const int width = min(dv - block_column, S::kColumns);
  T *y = static_cast<T *>(r.y);
  if (x.sequence >= w.cut.sequences) {  // behind the last sequence
    if constexpr (!kStates) {
      for (int64_t i = head_thread<kThreads>(); i < x.count * width; i += kThreads)
        y[((x.lo + x.at + i / width) * w.heads + head) * dv + block_column + i % width] =
            static_cast<T>(0.0f);
    }
    return;
  }
  if (kStates && x.last) return;

  const int lane = static_cast<int>(lane_id()), i = lane % 16, g = lane / 16;
  const int wave = kHeads > 1 ? 0 : static_cast<int>(wave_index());  // of the head
  // Column tile c of the block holds, of each 16 NT columns, those 4 in every kRun
  // that make neighbours of a lane's outputs: lane i's is part_of(c) + i / 4 kRun + i % 4.
  auto part_of = [](int c) { return c / NT * (16 * NT) + c % NT * 4; };
  const int64_t size = static_cast<int64_t>(dk) * dv;
  // The wave's state, state[kb][t][e]: row kb kFragment + g kRows + 4 t + e and the
  // lane's column of tile `wave`.  `visit` calls f(element, its address, whether it
  // exists); the address is a valid one in any case.
  f32x4 state[KB][kTiles] = {};
  const int row_of_lane = g * kRows;
  const int column_of_lane = block_column + part_of(wave) + i / 4 * kRun + i % 4;
  auto visit = [&](const float *base, int64_t which, bool transposed, auto f) {
    const char *p = reinterpret_cast<const char *>(base + (which * w.heads + head) * size);
    const uint32_t down = transposed ? 4 : 4 * dv, over = transposed ? 4 * dk : 4;
    const uint32_t offset = row_of_lane * down + column_of_lane * over;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = kb * kFragment + t * 4 + e;  // and the lane's
          const bool there = row + row_of_lane < dk && column_of_lane < dv;
          float value = state[kb][t][e];
          f(value, reinterpret_cast<const float *>(p + (there ? offset + row * down : 0u)), there);
          state[kb][t][e] = value;
        }
  };
  const float *begin = kStates ? nullptr : x.first ? r.initial : r.carried;
  if (begin != nullptr && dk > 0)
    visit(begin, x.first ? x.sequence : x.place - 1, r.transposed != 0,
          [&](float &value, const float *at, bool there) { value = there ? *at : 0.0f; });

  const float log2_decay = w.log_decay[head] * 1.44269504088896341f;
  const int early = r.early;
  // A wave's outputs: tiles first + own tiles of 16 tokens, of one part of the columns.
  constexpr int tiles = W < S::IT ? W : S::IT;
  const int first_tile = wave % tiles, part = wave / S::IT;
  // Weights of the pairs (i, j) of these tiles, with the scales; scores' rows are j,
  // their columns i.
  float weight[S::kOwn][JB][kPer], reach[S::kOwn];
  if constexpr (!kStates) {
#pragma unroll
    for (int own = 0; own < S::kOwn; ++own) {
      const int now = (first_tile + own * tiles) * 16 + i;
      reach[own] = r.scale_out * power(log2_decay, now + 1 - early);
#pragma unroll
      for (int b = 0; b < JB; ++b)
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const int apart = now - (b * kFragment + e / 4 * 16 + g * 4 + e % 4);
          weight[own][b][e] =
              apart >= 0 ? r.scale_in * r.scale_out * power(log2_decay, apart) : 0.0f;
        }
    }
  }
  // What is left at the end of a chunk of its tokens, and nothing of those behind
  // it: token j of `count` is at C - count + j.
  for (int j = head_thread<kThreads>(); j < 2 * C; j += kThreads)
    s_left[j] = j < C ? r.scale_in * power(log2_decay, C - 1 - j + early) : 0.0f;
  const float keep_all = power(log2_decay, C);

  // Token `t` of the walk is row lo + t of the inputs, or hi - 1 - t.
  const int64_t way = r.backwards != 0 ? -1 : 1;
  auto base_of = [&](const View &v) {
    const T *p = static_cast<const T *>(v.p) + head * v.head;
    p += w.cut.offsets == nullptr ? x.sequence * v.sequence : x.lo * v.token;
    return p + (r.backwards != 0 ? x.length - 1 - x.at : x.at) * v.token;
  };
  const int64_t q_step = way * r.q.token, k_step = way * r.k.token, v_step = way * r.v.token;
  const T *q_first = kStates ? nullptr : base_of(r.q), *k_first = base_of(r.k),
          *v_first = base_of(r.v) + block_column;
  Rows<T, KB, S::kOwn, kWhole> q_rows(q_step, dk);
  Stage<T, KD, C, kThreads, kWhole> k_stage(k_step, dk);
  Stage<T, S::kColumns, C, kThreads, kWhole> v_stage(v_step, width);
  auto load = [&](int64_t pos) {
    const int64_t rows = x.count - pos;
    k_stage.load(k_first + pos * k_step, k_step, rows);
    v_stage.load(v_first + pos * v_step, v_step, rows);
  };
  u32x4 q_raw[S::kOwn][KB];  // of the present chunk; q_rows those of the next
  auto load_q = [&](int64_t pos) {
    q_rows.load(q_first + pos * q_step, q_step, x.count - pos, first_tile, tiles);
  };
  // The wave's state as operands of its column tile.
  auto put_state = [&]() {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      float z[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) z[e] = state[kb][e / 4][e % 4];
      const Parts<U> parts = split<U>(z);
      char *p = s_s + ((kb * W + wave) * S::kOperands * 64 + lane) * 16;
      *reinterpret_cast<u32x4 *>(p) = parts.high;
      if constexpr (S::kOperands == 2) *reinterpret_cast<u32x4 *>(p + 1024) = parts.rest;
    }
  };

  // float32 products are dear: fragments past the channels of odd heads are left out
  // (3 heads of 33 x 45: 228 us forward and 247).
  auto none = [&](int kb) { return !kWhole && sizeof(T) == 4 && kb * kFragment >= dk; };

  if (head_thread<kThreads>() < 2) s_bad[head_thread<kThreads>()] = 0;
  load(0);
  if constexpr (!kStates) load_q(0);
  head_sync<kThreads>();
  int turn = 0;
  for (int64_t pos = 0; pos < x.count; turn ^= 1) {
    if constexpr (!kStates) {
      put_state();
      if (v_stage.bad()) s_bad[turn] = 1;
    }
    k_stage.put(s_k);
    v_stage.put(s_v);
    head_sync<kThreads>();
    int count = static_cast<int>(min(x.count - pos, static_cast<int64_t>(C)));
    if constexpr (!kStates) {
      if (s_bad[turn] != 0 && count > 1) {
        count = 1;
        clear_rows<T, KD, C, kThreads>(s_k);
        clear_rows<T, S::kColumns, C, kThreads>(s_v);
        head_sync<kThreads>();
      }
    }
    load(pos + count);
    if constexpr (!kStates) {
#pragma unroll
      for (int own = 0; own < S::kOwn; ++own)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) q_raw[own][kb] = q_rows.raw[own][kb];
      load_q(pos + count);
#pragma unroll
      for (int own = 0; own < S::kOwn; ++own) {
        const int it = first_tile + own * tiles;
        if (it * 16 >= count) break;
        f32x4 out[NT] = {};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          if (none(kb)) break;
          const Parts<U> q_parts = beside<T>(q_raw[own][kb]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const char *p = s_s + ((kb * W + part * NT + nt) * S::kOperands * 64 + lane) * 16;
            Parts<U> s_parts;
            s_parts.high = *reinterpret_cast<const u32x4 *>(p);
            if constexpr (S::kOperands == 2)
              s_parts.rest = *reinterpret_cast<const u32x4 *>(p + 1024);
            out[nt] = multiply_split<T, false>(q_parts, s_parts, out[nt]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) out[nt] *= reach[own];
#pragma unroll
        for (int b = 0; b < JB; ++b) {
          if (b * kTiles > it) break;
          float p[kPer];
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const int apart = it - b * kTiles - t;
            f32x4 score{0.0f, 0.0f, 0.0f, 0.0f};
            if (apart >= 0) {
#pragma unroll
              for (int kb = 0; kb < KB; ++kb) {
                if (none(kb)) break;
                score = multiply<T>(along<T, KD>(s_k, b * kFragment + t * 16 + i, kb * 4 + g),
                                    q_raw[own][kb], score);
              }
              if (apart == 0) {  // a later token's score may be anything
#pragma unroll
                for (int e = 0; e < 4; ++e) score[e] = i < g * 4 + e ? 0.0f : score[e];
              }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) p[t * 4 + e] = score[e] * weight[own][b][t * 4 + e];
          }
          const Parts<U> p_parts = split<U>(p);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const Parts<U> v_parts = beside<T>(
                across<T, S::kColumns, kRun>(s_v, b * kFragment, part_of(part * NT + nt)));
            out[nt] = multiply_split<T, true>(v_parts, p_parts, out[nt]);
          }
        }
        if (it * 16 + i < count) {
          // The tile's lowest row of y, and the lane's from there.
          const int64_t t = x.at + pos + it * 16;
          const int64_t token = x.lo + (r.backwards != 0 ? x.length - 16 - t : t);
          const int row = r.backwards != 0 ? 15 - i : i;
          const int column = block_column + part_of(part * NT) + g * kRun;
          const uint32_t offset = static_cast<uint32_t>(row * w.heads * dv + column) *
                                  static_cast<uint32_t>(sizeof(T));
          T *p = reinterpret_cast<T *>(
              reinterpret_cast<char *>(y + (token * w.heads + head) * dv) + offset);
          constexpr int kMost = 16 / static_cast<int>(sizeof(T)), kStore = kRun < kMost ? kRun : kMost;
#pragma unroll
          for (int c = 0; c < kRun; c += kStore) {
            Loose<T, kStore> z;
#pragma unroll
            for (int e = 0; e < kStore; ++e)
              z.v[e] = static_cast<T>(out[(c + e) / 4][(c + e) % 4]);
            if (column + c + kStore <= dv) {
              *reinterpret_cast<Loose<T, kStore> *>(p + c) = z;
            } else if (!kWhole || kRun < kMost) {
#pragma unroll
              for (int e = 0; e < kStore; ++e)
                if (column + c + e < dv) p[c + e] = z.v[e];
            }
          }
        }
      }
    }
    const float keep = count == C ? keep_all : power(log2_decay, count);
    Parts<U> fresh[JB];
#pragma unroll
    for (int b = 0; b < JB; ++b) {
      float z[kPer];
      widen<T>(across<T, S::kColumns, kRun>(s_v, b * kFragment, part_of(wave)), z);
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        z[e] *= s_left[C - count + b * kFragment + e / 4 * 16 + g * 4 + e % 4];
      fresh[b] = split<U, true>(z);
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        if (none(kb)) break;
        state[kb][t] *= keep;
#pragma unroll
        for (int b = 0; b < JB; ++b) {
          const Parts<U> k_parts =
              beside<T>(across<T, KD, kRows>(s_k, b * kFragment, kb * kFragment + t * 4));
          state[kb][t] = multiply_split<T, true, true>(k_parts, fresh[b], state[kb][t]);
        }
      }
    head_sync<kThreads>();
    if (head_thread<kThreads>() == 0) s_bad[turn] = 0;
    pos += count;
  }

  float *end = kStates ? r.carried : x.last ? r.final_state : nullptr;
  if (end == nullptr) return;
  if constexpr (kStates || W == 1) {
    visit(end, kStates ? x.place : x.sequence, false, [&](float &value, const float *at, bool there) {
      if (there) *const_cast<float *>(at) = value;
    });
  } else {
    // By LDS, as whole rows (2000 sequences of 17 tokens, 8 heads of 64 bfloat16: 154 us,
    // from the lanes 162).
    float *z = reinterpret_cast<float *>(s_s);
    static_assert(S::kS == KD * S::kColumns * 4, "the operands' room is the state's");
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          z[(kb * kFragment + row_of_lane + t * 4 + e) * S::kColumns + column_of_lane -
            block_column] = state[kb][t][e];
    head_sync<kThreads>();
    float *to = end + (x.sequence * w.heads + head) * size + block_column;
    constexpr int kWide = kWhole ? 4 : 1;  // floats of a store
    constexpr int kAcross = S::kColumns / kWide;
    const int column = head_thread<kThreads>() % kAcross * kWide;
    if (column < width) {
      for (int row = head_thread<kThreads>() / kAcross; row < dk; row += kThreads / kAcross) {
        Loose<float, kWide> out;
#pragma unroll
        for (int e = 0; e < kWide; ++e) out.v[e] = z[row * S::kColumns + column + e];
        *reinterpret_cast<Loose<float, kWide> *>(to + row * dv + column) = out;
      }
    }
  }
}

// One token of every sequence: the state is read, decayed, added to, stored and
// multiplied in one pass.  A block has one head of one sequence; its threads lie
// along the rows of the state, V columns each.  Bound by the state's bytes (64
// sequences, 8 heads of 64 x 64: 17 MB in 5.6 us, 3 TB/s) and, called, by the host.
template <typename T, int V>
__global__ __launch_bounds__(256) void decay_step_kernel(
    View q, View k, View v, const float *__restrict__ log_decay, const float *__restrict__ state,
    int64_t first, int heads, int dk, int dv, float scale, T *__restrict__ y,
    float *__restrict__ next) {
  __shared__ float s_q[kMostChannels], s_k[kMostChannels];
  __shared__ float s_sum[256 * V];
  const int64_t which = first + blockIdx.x, sequence = which / heads;
  const int head = static_cast<int>(which - sequence * heads);
  const T *qp = static_cast<const T *>(q.p) + sequence * q.token + head * q.head;
  const T *kp = static_cast<const T *>(k.p) + sequence * k.token + head * k.head;
  const T *vp = static_cast<const T *>(v.p) + sequence * v.token + head * v.head;
  if (static_cast<int>(threadIdx.x) < dk) {
    s_q[threadIdx.x] = static_cast<float>(qp[threadIdx.x]);
    s_k[threadIdx.x] = static_cast<float>(kp[threadIdx.x]);
  }
  const int across = (dv + V - 1) / V, rows = 256 / across;
  const int row0 = static_cast<int>(threadIdx.x) / across;
  const int column = (static_cast<int>(threadIdx.x) - row0 * across) * V;
  const float decay = expf(log_decay[head]);
  float fresh[V], sum[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    fresh[e] = row0 < rows ? static_cast<float>(vp[column + e]) : 0.0f;
    sum[e] = 0.0f;
  }
  __syncthreads();
  if (row0 < rows) {
    const int64_t base = which * dk * dv + column;
#pragma unroll 4
    for (int row = row0; row < dk; row += rows) {
      const int64_t at = base + static_cast<int64_t>(row) * dv;
      Pack<float, V> z = load_pack<float, V>(state + at);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        z.v[e] = fmaf(s_k[row], fresh[e], decay * z.v[e]);
        sum[e] = fmaf(s_q[row], z.v[e], sum[e]);
      }
      store_pack<float, V>(next + at, z);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) s_sum[row0 * dv + column + e] = sum[e];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < dv; c += 256) {
    float total = 0.0f;
    for (int i = 0; i < min(rows, dk); ++i) total += s_sum[i * dv + c];
    y[which * dv + c] = static_cast<T>(total * scale);
  }
}

// ---------------------------------------------------------------- host ----

struct Sizes {
  int type;
  bool ragged;
  int64_t sequences, length, n, heads, dk, dv;
};

// KD and W of a walk (see Shape): those of the wider of both heads' sides, which the
// backward's roles swap.
struct Form {
  int kd, waves;
  int columns() const { return 16 * waves; }
};
Form form_of(const Sizes &z) {
  const int64_t wide = std::max(z.dk, z.dv);
  if (wide <= 16) return {32, 1};
  if (wide <= 32) return {32, 2};
  return {wide <= 64 ? 64 : wide <= 128 ? 128 : 256, 4};
}

// Blocks of a walk that the device holds at once, by their registers and LDS.  A few
// blocks more would be a second round.
int64_t blocks_at_once(const Form &f) {
  return 256 * (f.waves == 1 ? 16 : f.waves == 2 ? 8 : f.kd == 64 ? 3 : f.kd == 128 ? 2 : 1);
}

// Tokens of a span: as many as fill the device once, but at least 256, so that a
// span's own tokens outweigh its states (200k tokens in 512 sequences, 4 heads of 64
// bfloat16, backward: 306 us, twice as many spans 357; 20k tokens in 40, 8 heads, spans
// of 128: 126, of 256: 98).
int64_t span_of(const Sizes &z) {
  const Form f = form_of(z);
  const int64_t blocks = std::max<int64_t>(1, z.heads * ceil_div(std::max(z.dk, z.dv), f.columns()));
  const int64_t longest = z.ragged ? z.n : z.length;
  const int64_t sequences = z.ragged ? 1 : std::max<int64_t>(1, z.sequences);
  const int64_t spans = std::max<int64_t>(1, blocks_at_once(f) / (blocks * sequences));
  const int64_t span = ceil_div(ceil_div(std::max<int64_t>(longest, 1), spans), 64) * 64;
  return std::max<int64_t>(256, span);
}

// Whether any sequence may have several spans, the number of states that they
// carry at most, and of items.
struct Plan {
  int64_t span, carried, items;
  int32_t spans;
  bool cut;
};
Plan plan_of(const Sizes &z) {
  Plan p{};
  p.span = span_of(z);
  if (z.ragged) {
    p.cut = z.n > p.span;
    p.carried = p.cut ? z.n / p.span : 0;
    p.items = z.sequences + 1 + (p.cut ? z.n / p.span + 1 : 0);
    p.spans = 1;
  } else {
    p.spans = static_cast<int32_t>(std::max<int64_t>(1, ceil_div(z.length, p.span)));
    p.cut = p.spans > 1;
    p.carried = z.sequences * (p.spans - 1);
    p.items = z.sequences * p.spans;
  }
  return p;
}

int64_t table_bytes(const Sizes &z, const Plan &p) {
  if (!z.ragged || !p.cut) return 0;
  Carver c(nullptr);
  c.take<int32_t>(p.items);
  c.take<int32_t>(p.carried);
  c.take<int32_t>(z.sequences + 2);
  return static_cast<int64_t>(align_up(c.used, 256));
}

template <typename T, int KD, int W, bool kStates, bool kWhole>
int launch_walk_as(Walk w, int64_t blocks, hipStream_t stream) {
  using S = Shape<T, KD, W, kStates>;
  constexpr int kLds = S::kLds * S::kHeads;
  static_assert(kLds + 2048 <= 160 * 1024, "LDS of a CU");
  if (kLds > 60 * 1024) {
    const hipError_t err = hipFuncSetAttribute(
        reinterpret_cast<const void *>(&decay_walk_kernel<T, KD, W, kStates, kWhole>),
        hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (err != hipSuccess) {
      set_error("decay_attention: %d bytes of LDS refused: %s", kLds, hipGetErrorString(err));
      return R2S_EHIP;
    }
  }
  constexpr int kBlock = 64 * W * S::kHeads;
  constexpr int64_t kMost = most_blocks(kBlock) / 8 * 8;  // whole turns of the XCDs
  for (int64_t first = 0; first < blocks; first += kMost) {
    w.first = static_cast<uint32_t>(first);
    decay_walk_kernel<T, KD, W, kStates, kWhole>
        <<<dim3(static_cast<uint32_t>(std::min(kMost, blocks - first))), dim3(kBlock), kLds,
           stream>>>(w);
    R2S_RETURN_IF(check_launch("decay_attention"));
  }
  return R2S_OK;
}
template <typename T, int KD, int W, bool kStates>
int launch_walk(const Walk &w, int64_t blocks, hipStream_t stream) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  return w.role[0].dk % kPer == 0 && w.role[0].dv % kPer == 0
             ? launch_walk_as<T, KD, W, kStates, true>(w, blocks, stream)
             : launch_walk_as<T, KD, W, kStates, false>(w, blocks, stream);
}

template <bool kStates>
int walk(const Sizes &z, const Plan &p, Walk &w, int roles, hipStream_t stream) {
  const Form f = form_of(z);
  int64_t columns = 0;
  for (int i = 0; i < roles; ++i)
    columns = std::max<int64_t>(columns, ceil_div(w.role[i].dv, f.columns()));
  w.column_blocks = static_cast<int32_t>(columns);
  w.roles = static_cast<uint32_t>(roles);
  const int64_t heads = f.waves == 1 ? ceil_div(z.heads, 4) : z.heads;
  int64_t blocks = p.items * heads * columns * roles;
  w.blocks = static_cast<uint32_t>(blocks);
  w.together = 0;
  if (z.ragged) {
    // All heads of an item, which may share lines; of few items, a head.
    const int64_t together = columns * roles * (p.items >= 64 ? heads : 1);
    w.together = static_cast<uint32_t>(together);
    blocks = together == 0 ? 0 : ceil_div(blocks, 8 * together) * 8 * together;
  }
  if (blocks > kInt32Max) {
    set_error("decay_attention: %lld blocks exceed 2^31 - 1", static_cast<long long>(blocks));
    return R2S_ERANGE;
  }
  if (blocks == 0) return R2S_OK;
  R2S_BY_TYPE(z.type, {
    if (f.waves == 1) return launch_walk<T, 32, 1, kStates>(w, blocks, stream);
    if (f.waves == 2) return launch_walk<T, 32, 2, kStates>(w, blocks, stream);
    if (f.kd == 64) return launch_walk<T, 64, 4, kStates>(w, blocks, stream);
    if (f.kd == 128) return launch_walk<T, 128, 4, kStates>(w, blocks, stream);
    return launch_walk<T, 256, 4, kStates>(w, blocks, stream);
  });
}

int carry(const Sizes &z, const Plan &p, const Walk &w, hipStream_t stream) {
  const int64_t states = z.heads * z.dk * z.dv, total = z.sequences * states;
  if (total == 0) return R2S_OK;
  if (!z.ragged && p.spans <= 16 && ceil_div(total, 256) <= kInt32Max) {
    decay_carry_few_kernel<<<dim3(static_cast<uint32_t>(ceil_div(total, 256))), dim3(256), 0,
                             stream>>>(w, total);
  } else {
    const int per = z.ragged ? 64 : 1;
    const int64_t rows = std::min<int64_t>(ceil_div(z.sequences, per), 65535);
    decay_carry_kernel<<<dim3(static_cast<uint32_t>(ceil_div(states, 64)),
                              static_cast<uint32_t>(rows)),
                         dim3(1024), 0, stream>>>(w, per);
  }
  return check_launch("decay_attention carry");
}

int check_sizes(const char *op, const Sizes &z) {
  R2S_REQUIRE(known_type(z.type), "%s: unknown element type %d", op, z.type);
  R2S_REQUIRE(z.sequences >= 0 && z.length >= 0 && z.n >= 0 && z.heads >= 0 && z.dk >= 0 &&
                  z.dv >= 0,
              "%s: negative size", op);
  if (z.dk > kMostChannels || z.dv > kMostChannels) {
    set_error("%s: at most %d channels of a head", op, kMostChannels);
    return R2S_ERANGE;
  }
  if (z.n > kInt32Max || z.sequences > kInt32Max - 2 || z.heads > 65535 || z.length > kInt32Max) {
    set_error("%s: at most 2^31 - 1 tokens and 65535 heads", op);
    return R2S_ERANGE;
  }
  if (z.ragged) {
    R2S_REQUIRE(z.sequences > 0 || z.n == 0, "%s: tokens without a sequence", op);
  } else {
    R2S_REQUIRE(z.sequences * z.length == z.n, "%s: %lld tokens are not %lld sequences of %lld",
                op, static_cast<long long>(z.n), static_cast<long long>(z.sequences),
                static_cast<long long>(z.length));
  }
  return R2S_OK;
}

bool bad_view(const Sizes &z, const View &v) {
  const __int128 reach = static_cast<__int128>(z.sequences) * v.sequence +
                         static_cast<__int128>(z.n) * v.token +
                         static_cast<__int128>(z.heads) * v.head;
  return v.sequence < 0 || v.token < 0 || v.token > kMostStep || v.head < 0 ||
         reach >= (static_cast<__int128>(1) << 60);
}

// The table of ragged items where sequences may have several spans.
int make_items(const Sizes &z, const Plan &p, Cut &cut, void *workspace, size_t bytes,
               hipStream_t stream) {
  const int64_t need = table_bytes(z, p);
  if (need == 0) return R2S_OK;
  if (workspace == nullptr || bytes < static_cast<size_t>(need)) {
    set_error("decay_attention: workspace of %zu bytes, %lld needed", bytes,
              static_cast<long long>(need));
    return R2S_EWORKSPACE;
  }
  Carver c(workspace);
  int32_t *order = c.take<int32_t>(p.items), *index = c.take<int32_t>(p.carried);
  int32_t *first = c.take<int32_t>(z.sequences + 2);
  cut.wholes = static_cast<int32_t>(p.carried);
  decay_items_kernel<<<dim3(1), dim3(1024), 0, stream>>>(cut, p.items, order, index, first);
  cut.order = order;
  cut.index = index;
  cut.first = first;
  return check_launch("decay_attention items");
}

Cut cut_of(const Sizes &z, const Plan &p, const int32_t *offsets) {
  Cut c{};
  c.offsets = offsets;
  c.n = z.n;
  c.sequences = z.sequences;
  c.length = z.length;
  c.span = p.span;
  c.carried = p.carried;
  c.spans = p.spans;
  return c;
}

}  // namespace
}  // namespace r2s

extern "C" {

int64_t r2s_decay_attention_kept_states(int32_t type, int32_t ragged, int64_t sequences,
                                        int64_t length, int64_t n, int64_t heads, int64_t dk,
                                        int64_t dv) {
  const r2s::Sizes z{type, ragged != 0, sequences, length, n, heads, dk, dv};
  if (r2s::check_sizes("decay_attention", z) != R2S_OK) return 0;
  return r2s::plan_of(z).carried;
}

int64_t r2s_decay_attention_workspace_bytes(int32_t type, int32_t ragged, int64_t sequences,
                                            int64_t length, int64_t n, int64_t heads, int64_t dk,
                                            int64_t dv, int32_t backward) {
  const r2s::Sizes z{type, ragged != 0, sequences, length, n, heads, dk, dv};
  if (r2s::check_sizes("decay_attention", z) != R2S_OK) return 0;
  const r2s::Plan p = r2s::plan_of(z);
  const int64_t states = backward != 0 ? p.carried * heads * dk * dv * 4 : 0;
  return r2s::table_bytes(z, p) + states;
}

int r2s_decay_attention_fwd(const void *q, int64_t q_sequence, int64_t q_token, int64_t q_head,
                            const void *k, int64_t k_sequence, int64_t k_token, int64_t k_head,
                            const void *v, int64_t v_sequence, int64_t v_token, int64_t v_head,
                            const float *log_decay, const float *initial, const int32_t *offsets,
                            int64_t sequences, int64_t length, int64_t n, int64_t heads,
                            int64_t dk, int64_t dv, float scale, int32_t type, int32_t reverse,
                            void *y, float *final_state, float *kept, void *workspace,
                            size_t workspace_bytes, r2s_stream_t st) {
  r2s::clear_error();
  const r2s::Sizes z{type, offsets != nullptr, sequences, length, n, heads, dk, dv};
  R2S_RETURN_IF(r2s::check_sizes("decay_attention_fwd", z));
  if (sequences == 0 || heads == 0 || (n == 0 && dk * dv == 0) || dv == 0) return R2S_OK;
  R2S_REQUIRE(log_decay != nullptr, "decay_attention_fwd: null decays");
  R2S_REQUIRE(dk == 0 || final_state != nullptr, "decay_attention_fwd: null final state");
  R2S_REQUIRE(n == 0 || (y != nullptr && (dk == 0 || (q != nullptr && k != nullptr)) &&
                         v != nullptr),
              "decay_attention_fwd: null tokens");
  r2s::Walk w{};
  r2s::Role &r = w.role[0];
  r.q = {q, q_sequence, q_token, q_head};
  r.k = {k, k_sequence, k_token, k_head};
  r.v = {v, v_sequence, v_token, v_head};
  R2S_REQUIRE(!r2s::bad_view(z, r.q) && !r2s::bad_view(z, r.k) && !r2s::bad_view(z, r.v),
              "decay_attention_fwd: bad stride");
  const r2s::Plan p = r2s::plan_of(z);
  R2S_REQUIRE(p.carried == 0 || dk == 0 || kept != nullptr,
              "decay_attention_fwd: null kept states");
  hipStream_t stream = r2s::as_stream(st);
  w.log_decay = log_decay;
  w.heads = static_cast<int32_t>(heads);
  w.cut = r2s::cut_of(z, p, offsets);
  R2S_RETURN_IF(r2s::make_items(z, p, w.cut, workspace, workspace_bytes, stream));
  r.initial = initial;
  r.carried = kept;
  r.dk = static_cast<int32_t>(dk);
  r.dv = static_cast<int32_t>(dv);
  r.backwards = reverse != 0;
  r.scale_in = 1.0f;
  r.scale_out = scale;
  r.y = y;
  r.final_state = final_state;
  if (p.cut && dk > 0) {
    R2S_RETURN_IF(r2s::walk<true>(z, p, w, 1, stream));
    R2S_RETURN_IF(r2s::carry(z, p, w, stream));
  }
  return r2s::walk<false>(z, p, w, 1, stream);
}

int r2s_decay_attention_bwd(const void *q, int64_t q_sequence, int64_t q_token, int64_t q_head,
                            const void *k, int64_t k_sequence, int64_t k_token, int64_t k_head,
                            const void *v, int64_t v_sequence, int64_t v_token, int64_t v_head,
                            const float *log_decay, const float *initial, const int32_t *offsets,
                            const float *kept, const void *v_y, int64_t vy_sequence,
                            int64_t vy_token, int64_t vy_head, const float *v_final,
                            int64_t sequences, int64_t length, int64_t n, int64_t heads,
                            int64_t dk, int64_t dv, float scale, int32_t type, int32_t reverse,
                            void *v_q, void *v_k, void *v_v, float *v_initial, void *workspace,
                            size_t workspace_bytes, r2s_stream_t st) {
  r2s::clear_error();
  const r2s::Sizes z{type, offsets != nullptr, sequences, length, n, heads, dk, dv};
  R2S_RETURN_IF(r2s::check_sizes("decay_attention_bwd", z));
  if (sequences == 0 || heads == 0 || dk == 0 || dv == 0) return R2S_OK;
  R2S_REQUIRE(log_decay != nullptr, "decay_attention_bwd: null decays");
  R2S_REQUIRE(n == 0 || (q && k && v && v_y && v_q && v_k && v_v),
              "decay_attention_bwd: null tokens");
  const r2s::View vq{q, q_sequence, q_token, q_head}, vk{k, k_sequence, k_token, k_head},
      vv{v, v_sequence, v_token, v_head}, vg{v_y, vy_sequence, vy_token, vy_head};
  R2S_REQUIRE(!r2s::bad_view(z, vq) && !r2s::bad_view(z, vk) && !r2s::bad_view(z, vv) &&
                  !r2s::bad_view(z, vg),
              "decay_attention_bwd: bad stride");
  const r2s::Plan p = r2s::plan_of(z);
  R2S_REQUIRE(p.carried == 0 || kept != nullptr, "decay_attention_bwd: null kept states");
  const int64_t table = r2s::table_bytes(z, p);
  const int64_t need = table + p.carried * heads * dk * dv * 4;
  if (need > 0 && (workspace == nullptr || workspace_bytes < static_cast<size_t>(need))) {
    r2s::set_error("decay_attention_bwd: workspace of %zu bytes, %lld needed", workspace_bytes,
                   static_cast<long long>(need));
    return R2S_EWORKSPACE;
  }
  hipStream_t stream = r2s::as_stream(st);
  r2s::Walk w{};
  w.log_decay = log_decay;
  w.heads = static_cast<int32_t>(heads);
  w.cut = r2s::cut_of(z, p, offsets);
  R2S_RETURN_IF(r2s::make_items(z, p, w.cut, workspace, workspace_bytes, stream));
  float *carried = reinterpret_cast<float *>(static_cast<char *>(workspace) + table);
  r2s::Role from_end{};  // R: what dk and dv have alike
  from_end.initial = v_final;
  from_end.carried = carried;
  from_end.backwards = reverse == 0;
  from_end.early = 1;
  from_end.scale_in = scale;
  from_end.scale_out = 1.0f;
  r2s::Role dv_role = from_end, dk_role = from_end, dq_role{};
  dv_role.q = vk;
  dv_role.k = vq;
  dv_role.v = vg;
  dv_role.dk = static_cast<int32_t>(dk);
  dv_role.dv = static_cast<int32_t>(dv);
  dv_role.y = v_v;
  dv_role.final_state = v_initial;
  dk_role.q = vv;
  dk_role.k = vg;
  dk_role.v = vq;
  dk_role.dk = static_cast<int32_t>(dv);
  dk_role.dv = static_cast<int32_t>(dk);
  dk_role.transposed = 1;
  dk_role.y = v_k;
  dq_role.q = vg;
  dq_role.k = vv;
  dq_role.v = vk;
  dq_role.initial = initial;
  dq_role.carried = const_cast<float *>(kept);  // read only: no states are made here
  dq_role.dk = static_cast<int32_t>(dv);
  dq_role.dv = static_cast<int32_t>(dk);
  dq_role.transposed = 1;
  dq_role.backwards = reverse != 0;
  dq_role.scale_in = 1.0f;
  dq_role.scale_out = scale;
  dq_role.y = v_q;
  w.role[0] = dv_role;
  if (p.cut) {
    R2S_RETURN_IF(r2s::walk<true>(z, p, w, 1, stream));
    R2S_RETURN_IF(r2s::carry(z, p, w, stream));
  }
  w.role[1] = dk_role;
  w.role[2] = dq_role;
  return r2s::walk<false>(z, p, w, 3, stream);
}

int r2s_decay_attention_step(const void *q, int64_t q_token, int64_t q_head, const void *k,
                             int64_t k_token, int64_t k_head, const void *v, int64_t v_token,
                             int64_t v_head, const float *log_decay, const float *state,
                             int64_t sequences, int64_t heads, int64_t dk, int64_t dv, float scale,
                             int32_t type, void *y, float *next, r2s_stream_t st) {
  r2s::clear_error();
  const r2s::Sizes z{type, false, sequences, 1, sequences, heads, dk, dv};
  R2S_RETURN_IF(r2s::check_sizes("decay_attention_step", z));
  if (sequences == 0 || heads == 0 || dv == 0) return R2S_OK;
  R2S_REQUIRE(log_decay && v && y && (dk == 0 || (q && k && state && next)),
              "decay_attention_step: null pointer");
  const r2s::View vq{q, 0, q_token, q_head}, vk{k, 0, k_token, k_head}, vv{v, 0, v_token, v_head};
  R2S_REQUIRE(!r2s::bad_view(z, vq) && !r2s::bad_view(z, vk) && !r2s::bad_view(z, vv),
              "decay_attention_step: bad stride");
  if (sequences * heads > r2s::kInt32Max) {
    r2s::set_error("decay_attention_step: more than 2^31 - 1 states");
    return R2S_ERANGE;
  }
  const bool wide = dv % 4 == 0 && (r2s::address(state) | r2s::address(next)) % 16 == 0;
  hipStream_t stream = r2s::as_stream(st);
  const int h = static_cast<int>(heads), a = static_cast<int>(dk), b = static_cast<int>(dv);
  constexpr int64_t kMost = r2s::most_blocks(256);
  for (int64_t first = 0; first < sequences * heads; first += kMost) {
    const dim3 grid(static_cast<uint32_t>(std::min(kMost, sequences * heads - first)));
    R2S_BY_TYPE(type, {
      if (wide)
        r2s::decay_step_kernel<T, 4><<<grid, dim3(256), 0, stream>>>(
            vq, vk, vv, log_decay, state, first, h, a, b, scale, static_cast<T *>(y), next);
      else
        r2s::decay_step_kernel<T, 1><<<grid, dim3(256), 0, stream>>>(
            vq, vk, vv, log_decay, state, first, h, a, b, scale, static_cast<T *>(y), next);
    });
    R2S_RETURN_IF(r2s::check_launch("decay_attention_step"));
  }
  return R2S_OK;
}

}  // extern "C"
