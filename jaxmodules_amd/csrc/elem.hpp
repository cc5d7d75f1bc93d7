// Chunks of V consecutive elements of a tensor as float: 16 bytes, or one element where
// lengths or addresses do not allow those.  Tag: bf16_tag, f16_tag or float.
#pragma once

#include <type_traits>

#include "common.hpp"

namespace mattn {

template <class Tag>
constexpr int kChunk = std::is_same_v<Tag, float> ? 4 : 8;

template <class Tag, int V>
__device__ __forceinline__ void load_v(const void* base, int64_t e, float (&o)[V]) {
  if constexpr (std::is_same_v<Tag, float>) {
    const float* p = (const float*)base + e;
    if constexpr (V % 4 == 0) {
#pragma unroll
      for (int j = 0; j < V / 4; ++j) {
        const f32x4 x = *(const f32x4*)(p + 4 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[4 * j + i] = x[i];
      }
    } else {
      static_assert(V == 1);
      o[0] = *p;
    }
  } else {
    const uint16_t* p = (const uint16_t*)base + e;
    if constexpr (V == 8) {
      const u32x4 x = *(const u32x4*)p;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = Elt<Tag>::to_f32(elt16(x, i));
    } else if constexpr (V == 4) {
      const u32x2 x = *(const u32x2*)p;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = Elt<Tag>::to_f32((x[i >> 1] >> (16 * (i & 1))) & 0xffffu);
    } else {
      static_assert(V == 1);
      o[0] = Elt<Tag>::to_f32(*p);
    }
  }
}

// The same as they lie in memory, and as float.
template <class Tag, int V>
using Raw = std::conditional_t<V == 1, std::conditional_t<std::is_same_v<Tag, float>, float, uint16_t>, u32x4>;
template <class Tag, int V>
__device__ __forceinline__ Raw<Tag, V> load_raw(const void* base, int64_t e) {
  return *(const Raw<Tag, V>*)((const char*)base + (std::is_same_v<Tag, float> ? 4 : 2) * e);
}
template <class Tag, int V>
__device__ __forceinline__ void from_raw(const Raw<Tag, V>& x, float (&o)[V]) {
  if constexpr (std::is_same_v<Tag, float>) {
    if constexpr (V == 1) {
      o[0] = x;
    } else {
      const f32x4 y = __builtin_bit_cast(f32x4, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = y[i];
    }
  } else if constexpr (V == 1) {
    o[0] = Elt<Tag>::to_f32(x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = Elt<Tag>::to_f32(elt16(x, i));
  }
}

template <class Tag, int V>
__device__ __forceinline__ void store_v(void* base, int64_t e, const float (&o)[V]) {
  if constexpr (std::is_same_v<Tag, float>) {
    float* p = (float*)base + e;
    if constexpr (V % 4 == 0) {
#pragma unroll
      for (int j = 0; j < V / 4; ++j) *(f32x4*)(p + 4 * j) = f32x4{o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]};
    } else {
      static_assert(V == 1);
      *p = o[0];
    }
  } else {
    uint16_t* p = (uint16_t*)base + e;
    if constexpr (V == 8) {
      *(u32x4*)p = u32x4{Elt<Tag>::pack2(o[0], o[1]), Elt<Tag>::pack2(o[2], o[3]), Elt<Tag>::pack2(o[4], o[5]),
                         Elt<Tag>::pack2(o[6], o[7])};
    } else if constexpr (V == 4) {
      *(u32x2*)p = u32x2{Elt<Tag>::pack2(o[0], o[1]), Elt<Tag>::pack2(o[2], o[3])};
    } else {
      static_assert(V == 1);
      *p = (uint16_t)(Elt<Tag>::pack2(o[0], 0.f) & 0xffffu);
    }
  }
}

}  // namespace mattn
