// Shared pieces of the latent decoder's operators (lookup.hip,
// gated_scan.hip, grouped.hip): element types, vectors of them, and the
// stable sort of ids that group.hip provides.
#pragma once

#include <initializer_list>

#include "r2s_common.h"

namespace r2s {

// Element types of activations, tables and weights; sums and states are
// float32 throughout.  float -> 16 bits rounds to nearest even.
using bf16_t = __bf16;
using f16_t = _Float16;

// V consecutive elements as one load or store.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T *p) {
  return *reinterpret_cast<const Pack<T, V> *>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, V> &x) {
  *reinterpret_cast<Pack<T, V> *>(p) = x;
}

inline int type_size(int type) { return type == R2S_TYPE_F32 ? 4 : 2; }
inline bool known_type(int type) {
  return type == R2S_TYPE_F32 || type == R2S_TYPE_BF16 || type == R2S_TYPE_F16;
}

inline uint64_t address(const void *p) { return reinterpret_cast<uint64_t>(p); }

// Stable grouping of n ids by value (group.hip): order [n] receives the
// positions sorted by (id, position), ids outside [0, n_groups) last; keys [n]
// (may be null) the sorted ids, n_groups for those outside; offsets
// [n_groups + 1] (may be null) each group's first index in order,
// offsets[n_groups] the number of ids inside.
int64_t sort_ids_bytes(int64_t n, int64_t n_groups);
int sort_ids(const void *ids, bool wide, int64_t n, int64_t n_groups, int32_t *order,
             int32_t *offsets, uint32_t *keys, void *workspace, hipStream_t stream);

// The expression `call` with T bound to the element type.
#define R2S_BY_TYPE(type, ...)                   \
  do {                                           \
    if ((type) == R2S_TYPE_F32) {                \
      using T = float;                           \
      __VA_ARGS__;                               \
    } else if ((type) == R2S_TYPE_BF16) {        \
      using T = ::r2s::bf16_t;                   \
      __VA_ARGS__;                               \
    } else {                                     \
      using T = ::r2s::f16_t;                    \
      __VA_ARGS__;                               \
    }                                            \
  } while (0)

}  // namespace r2s
