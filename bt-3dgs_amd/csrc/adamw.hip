// AdamW (decoupled weight decay) over many tensors in one launch for every 32:
//
//   p *= 1 - lr wd,  m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p -= lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps).
//
// Parameters and gradients are float32, bfloat16 or float16; a 16-bit parameter
// has a float32 master copy that the step is made on, and is its rounding after it.
// Where the parameter is something else before the step, it was written in between
// (a checkpoint, a clamp), and the step goes on from that value.  The
// states are float32, or 8 bits: float8 (e4m3) codes of m and of sqrt(v), each run
// of 256 elements with a float32 scale that takes its largest element to 448.  The
// root has half the exponent range of v, which e4m3's 2^18 covers; a nonzero one is
// never rounded to zero, as the step divides by it.  A code is rounded up with the
// probability of the fraction that is cut off: to nearest, an average that moves by
// less than half a code a step (b2 = 0.99 moves v by 1 % at most where codes lie 6
// to 12 % apart) would never move.  The chances are a hash of the element's index
// and the step, so a step can be made again bit for bit.  An element that is not
// finite becomes a NaN and is left out of its run's scale.
//
// One wave steps one run of 256 elements, four neighbours a lane, so that every
// array moves in whole lines and the run's largest element is a reduction over the
// wave; a block takes 16 runs of one tensor.  Tensors lie one behind another in
// the grid, so small ones cost a block each and not a column of the largest's.
// Bound by the bytes: 16 per float32 element with 8-bit states, 28 with float32 ones,
// of 16-bit parameters 18 and 30 (two tables of 200k x 256 float32, 8-bit states: 1.65
// GB in 314 to 316 us, 5.2 TB/s; the 76 tensors of twelve bfloat16 blocks of 512
// channels, three launches: 1.56 GB in 336, 4.6 TB/s, two bytes of an element for
// reading the parameters to see what was written to them).
#include <algorithm>

#include "r2s_latent.h"

namespace r2s {
namespace {

constexpr int kThreads = 256;
constexpr int kRun = 256;           // elements of a scale: four for each lane of a wave
constexpr int kRunsPerWave = 4;
constexpr int kPerBlock = kRun * kRunsPerWave * (kThreads / 64);
constexpr int kMostTensors = 32;    // of a launch
constexpr int64_t kMostBlocks = most_blocks(kThreads);
constexpr float kMostCode = 448.0f, kLeastCode = 0x1p-9f, kLeastNormal = 0x1p-6f;

struct AdamwTable {
  r2s_adamw_tensor_t t[kMostTensors];
  uint32_t first[kMostTensors + 1];  // each tensor's first block
  int32_t count;
};

// The chance of element i at this step: 32 bits of which the mean and the root
// take 16 each.  The multipliers are the fractions of the square roots of 2 and 3,
// made odd; the step's is that of the golden ratio.
__device__ __forceinline__ uint32_t chance(uint32_t i, uint32_t step) {
  uint32_t h = i + step * 0x9E3779B9u;
  h ^= h >> 16;
  h *= 0x6A09E667u;
  h ^= h >> 15;
  h *= 0xBB67AE85u;
  return h ^ (h >> 16);
}

// |x| in code units (at most 448) with the bits below a code's step cut off, after
// r / 2^16 of a step was added.  Adding to the float's bits carries into the
// exponent as the codes do.
__device__ __forceinline__ float cut(float y, uint32_t r) {
  const float normal = __uint_as_float((__float_as_uint(y) + (r << 4)) & 0xFFF00000u);
  const float small =
      floorf(fmaf(y, 512.0f, static_cast<float>(r) * 0x1p-16f)) * kLeastCode;
  return fminf(y < kLeastNormal ? small : normal, kMostCode);
}

__device__ __forceinline__ float wave_max(float v) {
  return __uint_as_float(r2s::wave_max(__float_as_uint(v)));  // not negative: ordered as bits
}

__device__ __forceinline__ bool finite(float x) {
  return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u;
}

__device__ __forceinline__ bool same_bits(float a, float b) {
  return __float_as_uint(a) == __float_as_uint(b);
}

// Four float8 codes <-> floats that are codes' values.
__device__ __forceinline__ void decode(uint32_t c, float (&x)[4]) {
  x[0] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c), 0);
  x[1] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c), 1);
  x[2] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c), 2);
  x[3] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c), 3);
}
__device__ __forceinline__ uint32_t encode(const float (&x)[4]) {
  int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], c, true));
}

// Codes of x, whose scale is stored at `scale` by one lane.
template <bool kRoot>
__device__ __forceinline__ uint32_t quantize(const float (&x)[4], const uint32_t (&r)[4],
                                             float *scale) {
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) most = fmaxf(most, finite(x[i]) ? fabsf(x[i]) : 0.0f);
  const float s = fmaxf(__fmul_rn(wave_max(most), 1.0f / kMostCode), 0x1p-126f);
  if (lane_id() == 0) *scale = s;
  const float inverse = 1.0f / s;
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float c = cut(fminf(fabsf(x[i]) * inverse, kMostCode),
                  kRoot ? r[i] >> 16 : r[i] & 0xFFFFu);
    if (kRoot && x[i] > 0.0f) c = fmaxf(c, kLeastCode);
    y[i] = finite(x[i]) ? copysignf(c, x[i]) : __builtin_nanf("");
  }
  return encode(y);
}

// Four elements from i on, of n: 4 sizeof(T) bytes at once where the array is
// aligned, else one after the other.
template <typename T>
__device__ __forceinline__ void load4(const void *p, int64_t i, int64_t n, bool vec,
                                      float (&x)[4]) {
  const T *at = static_cast<const T *>(p) + i;
  if (vec && i + 4 <= n) {
    const Pack<T, 4> v = load_pack<T, 4>(at);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = static_cast<float>(v.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = i + j < n ? static_cast<float>(at[j]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void store4(void *p, int64_t i, int64_t n, bool vec,
                                       const float (&x)[4]) {
  T *at = static_cast<T *>(p) + i;
  if (vec && i + 4 <= n) {
    Pack<T, 4> v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v.v[j] = static_cast<T>(x[j]);
    store_pack<T, 4>(at, v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) at[j] = static_cast<T>(x[j]);
  }
}
__device__ __forceinline__ uint32_t load_codes(const void *p, int64_t i, int64_t n, bool vec) {
  const uint8_t *at = static_cast<const uint8_t *>(p) + i;
  if (vec && i + 4 <= n) return *reinterpret_cast<const uint32_t *>(at);
  uint32_t c = 0;
  for (int j = 0; j < 4; ++j)
    if (i + j < n) c |= static_cast<uint32_t>(at[j]) << (8 * j);
  return c;
}
__device__ __forceinline__ void store_codes(void *p, int64_t i, int64_t n, bool vec, uint32_t c) {
  uint8_t *at = static_cast<uint8_t *>(p) + i;
  if (vec && i + 4 <= n) {
    *reinterpret_cast<uint32_t *>(at) = c;
  } else {
    for (int j = 0; j < 4; ++j)
      if (i + j < n) at[j] = static_cast<uint8_t>(c >> (8 * j));
  }
}

// The roundings of the float32 step are those of torch's element-wise AdamW: each
// product, quotient and sum on its own, lerp and the two multiply-adds fused.
__device__ __forceinline__ void step32(const r2s_adamw_tensor_t &d, float &p, float g, float &m,
                                       float &v) {
  p = __fmul_rn(p, d.keep);
  const float diff = g - m;
  m = d.lerp_weight < 0.5f ? fmaf(d.lerp_weight, diff, m)
                           : fmaf(-diff, 1.0f - d.lerp_weight, g);
  v = fmaf(d.one_minus_beta2, __fmul_rn(g, g), __fmul_rn(v, d.beta2));
  const float den = __fadd_rn(__fdiv_rn(sqrtf(v), d.bias_correction2_sqrt), d.eps);
  p = fmaf(d.step_size, __fdiv_rn(m, den), p);
}

// The averages of a step from codes, every product, sum and root rounded on its
// own: a code next to where its chance cuts hangs on the last bit, and this way it
// is that of the elementary operations however the compiler would join them.
__device__ __forceinline__ void step8(const r2s_adamw_tensor_t &d, float m_scale, float r_scale,
                                      float g, float &m, float &r) {
#pragma clang fp contract(off)
  m = m * m_scale;
  m = d.beta1 * m + d.lerp_weight * g;
  r = r * r_scale;
  const float square = d.beta2 * r * r + d.one_minus_beta2 * g * g;
  if (square == __builtin_inff()) {  // the squares' sum, or an infinite gradient's root too
    const float small = r * 0x1p-66f, g_small = g * 0x1p-66f;
    r = sqrtf(d.beta2 * small * small + d.one_minus_beta2 * g_small * g_small) * 0x1p66f;
  } else {
    r = sqrtf(square);
  }
}

template <typename T, bool k8>
__device__ __forceinline__ void step_runs(const r2s_adamw_tensor_t &d, int64_t base) {
  // Every array at a multiple of its four elements' bytes.
  const uint64_t wide = address(d.master) | (sizeof(T) == 4 ? address(d.param) | address(d.grad) : 0) |
                        (k8 ? 0 : address(d.exp_avg) | address(d.second));
  const uint64_t half = sizeof(T) == 2 ? address(d.param) | address(d.grad) : 0;
  const uint64_t codes = k8 ? address(d.exp_avg) | address(d.second) : 0;
  const bool vec = wide % 16 == 0 && half % 8 == 0 && codes % 4 == 0;
  void *master = d.master != nullptr ? static_cast<void *>(d.master) : d.param;
  const float root_correction = 1.0f / d.bias_correction2_sqrt;
#pragma unroll 2
  for (int run = 0; run < kRunsPerWave; ++run) {
    const int64_t start = base + run * kRun;  // wave-uniform
    if (start >= d.n) return;
    const int64_t i = start + static_cast<int>(lane_id()) * 4;
    float p[4], g[4], m[4], v[4];
    load4<T>(d.grad, i, d.n, vec, g);
    load4<float>(master, i, d.n, vec, p);
    if constexpr (sizeof(T) == 2) {
      float now[4];  // what the copy rounds to, or what was written since
      load4<T>(d.param, i, d.n, vec, now);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        p[j] = same_bits(static_cast<float>(static_cast<T>(p[j])), now[j]) ? p[j] : now[j];
    }
    if constexpr (!k8) {
      load4<float>(d.exp_avg, i, d.n, vec, m);
      load4<float>(d.second, i, d.n, vec, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) step32(d, p[j], g[j], m[j], v[j]);
      store4<float>(d.exp_avg, i, d.n, vec, m);
      store4<float>(d.second, i, d.n, vec, v);
    } else {
      const uint32_t mc = load_codes(d.exp_avg, i, d.n, vec);
      const uint32_t rc = load_codes(d.second, i, d.n, vec);
      const int64_t at = start / kRun;
      const float ms = d.exp_avg_scale[at], rs = d.second_scale[at];
      decode(mc, m);
      decode(rc, v);
      uint32_t r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        step8(d, ms, rs, g[j], m[j], v[j]);
        p[j] = fmaf(d.step_size * m[j],
                    __builtin_amdgcn_rcpf(fmaf(v[j], root_correction, d.eps)), p[j] * d.keep);
        r[j] = chance(static_cast<uint32_t>(i + j), d.step);
      }
      store_codes(d.exp_avg, i, d.n, vec, quantize<false>(m, r, d.exp_avg_scale + at));
      store_codes(d.second, i, d.n, vec, quantize<true>(v, r, d.second_scale + at));
    }
    store4<float>(master, i, d.n, vec, p);
    if constexpr (sizeof(T) == 2) store4<T>(d.param, i, d.n, vec, p);
  }
}

template <bool k8>
__device__ __forceinline__ void step_by_type(const r2s_adamw_tensor_t &d, int64_t base) {
  if (d.type == R2S_TYPE_F32)
    step_runs<float, k8>(d, base);
  else if (d.type == R2S_TYPE_BF16)
    step_runs<bf16_t, k8>(d, base);
  else
    step_runs<f16_t, k8>(d, base);
}

__global__ __launch_bounds__(kThreads) void adamw_kernel(AdamwTable table) {
  int at = 0;  // the last tensor whose first block is not past this one
  for (int step = kMostTensors / 2; step > 0; step /= 2)
    if (at + step < table.count && table.first[at + step] <= blockIdx.x) at += step;
  const r2s_adamw_tensor_t &d = table.t[at];
  const int64_t base = static_cast<int64_t>(blockIdx.x - table.first[at]) * kPerBlock +
                       static_cast<int64_t>(wave_index()) * (kRun * kRunsPerWave);
  if (base >= d.n) return;
  if (d.exp_avg_scale != nullptr)
    step_by_type<true>(d, base);
  else
    step_by_type<false>(d, base);
}

}  // namespace
}  // namespace r2s

extern "C" {

int r2s_adamw_step(const r2s_adamw_tensor_t *tensors, int32_t n_tensors, r2s_stream_t st) {
  r2s::clear_error();
  R2S_REQUIRE(n_tensors >= 0 && (n_tensors == 0 || tensors != nullptr),
              "adamw_step: bad tensor list");
  for (int32_t i = 0; i < n_tensors; ++i) {
    const r2s_adamw_tensor_t &t = tensors[i];
    R2S_REQUIRE(t.n >= 0, "adamw_step: tensor %d has a negative size", i);
    R2S_REQUIRE(r2s::known_type(t.type), "adamw_step: tensor %d has element type %d", i, t.type);
    if (t.n == 0) continue;
    R2S_REQUIRE(t.param && t.grad && t.exp_avg && t.second,
                "adamw_step: tensor %d has a null pointer", i);
    R2S_REQUIRE((t.type == R2S_TYPE_F32) == (t.master == nullptr),
                "adamw_step: tensor %d: 16-bit parameters have a master, float32 ones none", i);
    R2S_REQUIRE((t.exp_avg_scale == nullptr) == (t.second_scale == nullptr),
                "adamw_step: tensor %d has one scale of two", i);
    if (t.n > r2s::kMostBlocks * r2s::kPerBlock) {
      r2s::set_error("adamw_step: tensor %d is too large: more than %lld elements", i,
                     static_cast<long long>(r2s::kMostBlocks * r2s::kPerBlock));
      return R2S_ERANGE;
    }
  }
  for (int32_t next = 0; next < n_tensors;) {
    r2s::AdamwTable table{};
    int64_t blocks = 0;
    for (; next < n_tensors && table.count < r2s::kMostTensors; ++next) {
      const int64_t more = r2s::ceil_div(tensors[next].n, r2s::kPerBlock);
      if (more == 0) continue;
      if (blocks + more > r2s::kMostBlocks) break;
      table.t[table.count] = tensors[next];
      table.first[table.count++] = static_cast<uint32_t>(blocks);
      blocks += more;
    }
    if (table.count == 0) continue;
    r2s::adamw_kernel<<<dim3(static_cast<uint32_t>(blocks)), dim3(r2s::kThreads), 0,
                        r2s::as_stream(st)>>>(table);
    R2S_RETURN_IF(r2s::check_launch("adamw_step"));
  }
  return R2S_OK;
}

}  // extern "C"
