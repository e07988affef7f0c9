// Rotary positions along several axes.  A head's first 2 R channels are R pairs;
// pair j belongs to one axis and has its frequency,
//
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position[axis] freq_j,
//   freq_j = base^(-i / m),
//
// with i the pair's number within its axis' m pairs, or (shared) within all R;
// the channels behind the pairs are copied.  The gradient is the same turn the
// other way.
//
// Angles are products in 64 bits, of which only the part of a turn goes on in
// 32: a position of 10^6 in 32 bits is off by 0.03 rad and more.  Every head of a
// token has the same angles, so a block computes those of a few tokens into LDS
// first; then its threads walk the tokens' heads in the order of memory, 16 bytes
// of each half of the pairs at a time.  Bound by the bytes: both tensors are read
// and written once (32k tokens, q of 16 heads and k of 4 of 64 bfloat16: 168 MB in
// 40 to 43 us, 3.9 to 4.2 TB/s); 64 tokens take 3.5 us, the launch's own.
#include <algorithm>

#include "r2s_latent.h"

namespace r2s {
namespace {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryPairs = 1024;  // cosines and sines of a block: 8 KB of LDS

struct RotaryPlan {
  int32_t axes, pairs, head;  // axes, R, channels of a head
  int32_t shared, interleaved;
  int32_t sections[R2S_ROTARY_MAX_AXES];
  double log2_base;
  float sign;  // -1 turns back
};

// One tensor: heads of a token and of all tokens by strides, the output dense.
struct RotaryTensor {
  const void *in;
  void *out;
  int64_t token_stride, head_stride;
  int32_t heads;
};

// V elements at any element.
template <typename T, int V>
struct __attribute__((packed)) Loose {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void turn(const Loose<T, V> &a, const Loose<T, V> &b,
                                     const float2 *__restrict__ wheel, Loose<T, V> &x,
                                     Loose<T, V> &y) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float2 w = wheel[i];
    const float p = static_cast<float>(a.v[i]), q = static_cast<float>(b.v[i]);
    x.v[i] = static_cast<T>(fmaf(p, w.x, -(q * w.y)));
    y.v[i] = static_cast<T>(fmaf(q, w.x, p * w.y));
  }
}

__device__ __forceinline__ double position(const void *p, int type, int64_t i) {
  if (type == R2S_POSITION_F32) return static_cast<const float *>(p)[i];
  if (type == R2S_POSITION_I32) return static_cast<const int32_t *>(p)[i];
  return static_cast<double>(static_cast<const int64_t *>(p)[i]);
}

// V: pairs of a thread (one where a head has fewer than a vector of them).  A
// last vector ends with the pairs and overlaps the one before it.
template <typename T, int V>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(
    RotaryTensor q, RotaryTensor k, RotaryPlan plan, const void *__restrict__ positions,
    int position_type, int64_t before, int64_t n, int tokens) {
  __shared__ float2 s_wheel[kRotaryPairs];
  const int64_t first = before + static_cast<int64_t>(blockIdx.x) * tokens;
  const int here = static_cast<int>(min(static_cast<int64_t>(tokens), n - first));
  const int pairs = plan.pairs;
  for (int i = threadIdx.x; i < here * pairs; i += kRotaryThreads) {
    const int token = i / pairs, pair = i - token * pairs;
    int axis = 0, index = pair;
    while (axis + 1 < plan.axes && index >= plan.sections[axis]) index -= plan.sections[axis++];
    const double rate = plan.shared != 0
                            ? static_cast<double>(pair) / pairs
                            : static_cast<double>(index) / plan.sections[axis];
    const double turns = position(positions, position_type, (first + token) * plan.axes + axis) *
                         (exp2(-rate * plan.log2_base) * 0.15915494309189533577);
    float sine, cosine;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sine, &cosine);
    s_wheel[i] = make_float2(cosine, plan.sign * sine);
  }
  __syncthreads();
  const int rest = plan.head - 2 * pairs;
  const int turned = (pairs + V - 1) / V, items = turned + (rest + V - 1) / V;
  const int heads = q.heads + k.heads;
  for (int i = threadIdx.x; i < here * heads * items; i += kRotaryThreads) {
    const int row = i / items, item = i - row * items;
    const int token = row / heads, slot = row - token * heads;
    const bool of_q = slot < q.heads;
    const int head = of_q ? slot : slot - q.heads;
    const T *in = static_cast<const T *>(of_q ? q.in : k.in) +
                  (first + token) * (of_q ? q.token_stride : k.token_stride) +
                  head * (of_q ? q.head_stride : k.head_stride);
    T *out = static_cast<T *>(of_q ? q.out : k.out) +
             ((first + token) * (of_q ? q.heads : k.heads) + head) * plan.head;
    if (item < turned) {
      const int j = min(item * V, pairs - V);
      const float2 *wheel = s_wheel + token * pairs + j;
      if (plan.interleaved != 0) {
        const Loose<T, 2 * V> z = *reinterpret_cast<const Loose<T, 2 * V> *>(in + 2 * j);
        Loose<T, V> a, b, x, y;
#pragma unroll
        for (int e = 0; e < V; ++e) a.v[e] = z.v[2 * e], b.v[e] = z.v[2 * e + 1];
        turn<T, V>(a, b, wheel, x, y);
        Loose<T, 2 * V> w;
#pragma unroll
        for (int e = 0; e < V; ++e) w.v[2 * e] = x.v[e], w.v[2 * e + 1] = y.v[e];
        *reinterpret_cast<Loose<T, 2 * V> *>(out + 2 * j) = w;
      } else {
        const Loose<T, V> a = *reinterpret_cast<const Loose<T, V> *>(in + j);
        const Loose<T, V> b = *reinterpret_cast<const Loose<T, V> *>(in + pairs + j);
        Loose<T, V> x, y;
        turn<T, V>(a, b, wheel, x, y);
        *reinterpret_cast<Loose<T, V> *>(out + j) = x;
        *reinterpret_cast<Loose<T, V> *>(out + pairs + j) = y;
      }
    } else {
      const int j = 2 * pairs + (item - turned) * V;
      for (int e = j; e < min(j + V, plan.head); ++e) out[e] = in[e];
    }
  }
}

template <typename T, int V>
int launch_rotary(const RotaryTensor &q, const RotaryTensor &k, const RotaryPlan &plan,
                  const void *positions, int position_type, int64_t n, hipStream_t stream) {
  // As many tokens as fill the threads eight times, but enough blocks for the
  // device, and no more than LDS has room for.
  const int64_t items = static_cast<int64_t>(q.heads + k.heads) * ((plan.head + 2 * V - 1) / (2 * V));
  int64_t tokens = std::max<int64_t>(1, 8 * kRotaryThreads / std::max<int64_t>(items, 1));
  tokens = std::min<int64_t>(tokens, std::max<int64_t>(1, n / 1024));
  tokens = std::min<int64_t>(tokens, std::max(1, kRotaryPairs / std::max(plan.pairs, 1)));
  const int64_t blocks = ceil_div(n, tokens), most = most_blocks(kRotaryThreads);
  for (int64_t b = 0; b < blocks; b += most) {
    rotary_kernel<T, V><<<dim3(static_cast<uint32_t>(std::min(most, blocks - b))),
                          dim3(kRotaryThreads), 0, stream>>>(
        q, k, plan, positions, position_type, b * tokens, n, static_cast<int>(tokens));
    R2S_RETURN_IF(check_launch("rotary_axes"));
  }
  return R2S_OK;
}

// The largest element of a tensor that is read, and whether it fits an address.
bool reach_fits(int64_t n, int64_t token_stride, int64_t heads, int64_t head_stride) {
  const __int128 last = static_cast<__int128>(n) * token_stride +
                        static_cast<__int128>(heads) * head_stride;
  return last < (static_cast<__int128>(1) << 60);
}

}  // namespace
}  // namespace r2s

extern "C" {

int r2s_rotary_axes(const void *q, int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads,
                    const void *k, int64_t k_token_stride, int64_t k_head_stride, int64_t k_heads,
                    const void *positions, int32_t position_type, const int32_t *sections,
                    int32_t axes, int32_t shared, double base, int32_t interleaved,
                    int32_t inverse, int32_t type, int64_t n, int64_t head, void *q_out,
                    void *k_out, r2s_stream_t st) {
  r2s::clear_error();
  R2S_REQUIRE(r2s::known_type(type), "rotary_axes: unknown element type %d", type);
  R2S_REQUIRE(n >= 0 && q_heads >= 0 && k_heads >= 0 && head >= 0, "rotary_axes: negative size");
  R2S_REQUIRE(position_type >= R2S_POSITION_F32 && position_type <= R2S_POSITION_I64,
              "rotary_axes: unknown position type %d", position_type);
  R2S_REQUIRE(axes >= 1 && axes <= R2S_ROTARY_MAX_AXES, "rotary_axes: 1 to %d axes, got %d",
              R2S_ROTARY_MAX_AXES, axes);
  R2S_REQUIRE(sections != nullptr, "rotary_axes: null sections");
  R2S_REQUIRE(base > 0.0 && base < 1e300, "rotary_axes: base must be positive and finite");
  r2s::RotaryPlan plan{};
  int64_t pairs = 0;
  for (int a = 0; a < axes; ++a) {
    R2S_REQUIRE(sections[a] >= 0, "rotary_axes: section %d is negative", a);
    plan.sections[a] = sections[a];
    pairs += sections[a];
  }
  R2S_REQUIRE(2 * pairs <= head, "rotary_axes: %lld pairs do not fit a head of %lld channels",
              static_cast<long long>(pairs), static_cast<long long>(head));
  const int64_t heads = q_heads + k_heads;
  if (n > r2s::kInt32Max || heads > 65535 || head > 2048) {
    r2s::set_error("rotary_axes: at most 2^31 - 1 tokens, 65535 heads and 2048 channels");
    return R2S_ERANGE;
  }
  if (n == 0 || heads == 0 || head == 0) return R2S_OK;
  R2S_REQUIRE(positions != nullptr, "rotary_axes: null positions");
  R2S_REQUIRE(q_heads == 0 || (q != nullptr && q_out != nullptr), "rotary_axes: null q");
  R2S_REQUIRE(k_heads == 0 || (k != nullptr && k_out != nullptr), "rotary_axes: null k");
  R2S_REQUIRE(q_token_stride >= 0 && q_head_stride >= 0 && k_token_stride >= 0 &&
                  k_head_stride >= 0 && r2s::reach_fits(n, q_token_stride, q_heads, q_head_stride) &&
                  r2s::reach_fits(n, k_token_stride, k_heads, k_head_stride),
              "rotary_axes: bad stride");
  plan.axes = axes;
  plan.pairs = static_cast<int32_t>(pairs);
  plan.head = static_cast<int32_t>(head);
  plan.shared = shared != 0;
  plan.interleaved = interleaved != 0;
  plan.log2_base = log2(base);
  plan.sign = inverse != 0 ? -1.0f : 1.0f;
  const r2s::RotaryTensor tq{q, q_out, q_token_stride, q_head_stride,
                             static_cast<int32_t>(q_heads)};
  const r2s::RotaryTensor tk{k, k_out, k_token_stride, k_head_stride,
                             static_cast<int32_t>(k_heads)};
  hipStream_t stream = r2s::as_stream(st);
  R2S_BY_TYPE(type, {
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    if (pairs >= V)
      return r2s::launch_rotary<T, V>(tq, tk, plan, positions, position_type, n, stream);
    return r2s::launch_rotary<T, 1>(tq, tk, plan, positions, position_type, n, stream);
  });
}

}  // extern "C"
