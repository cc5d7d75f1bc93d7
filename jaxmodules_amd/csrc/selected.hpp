// Operands of the selected-attention kernels: MFMA fragments, tiles in LDS and their
// reads, for 16-bit inputs (32x32x16 and 16x16x32 products) and float32 (the same depth
// as eight 32x32x2 or 16x16x4 products, so that all layouts are shared).
//
// 32x32: lane l = 32 hi + l32 holds A row l32 / B column l32 at k = 8 hi .. 8 hi + 7, and
// of the result column l32, rows 8 (r / 4) + 4 hi + r % 4 in register r.  Registers
// 8 j .. 8 j + 7 of a result are the B operand of the next product over rows 16 j ..
// 16 j + 15, slot e standing for row 16 j + 8 (e / 4) + 4 hi + e % 4 (tr_frag reads its
// A operand in the same order).
// 16x16: lane 16 g + l16, k = 8 g .. 8 g + 7; result rows 4 g + r.  Two 16-row results
// are the B operand of a 32-deep product, slots 0-3 rows 4 g + e of the first, 4-7 of
// the second.
#pragma once

#include "elem.hpp"

namespace mattn {

struct F8 {  // eight float32 values, one operand of a 16- or 32-deep step
  f32x4 a, b;
};

template <class Tag>
struct SOp {  // 16-bit
  using Frag = u32x4;
  static constexpr int ES = 2;
  static __device__ __forceinline__ f32x16 mma32(const Frag& a, const Frag& b, f32x16 c) { return Elt<Tag>::mfma(a, b, c); }
  static __device__ __forceinline__ f32x4 mma16(const Frag& a, const Frag& b, f32x4 c) {
    if constexpr (std::is_same_v<Tag, bf16_tag>)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ Frag pack(const float (&x)[8]) {
    return Frag{Elt<Tag>::pack2(x[0], x[1]), Elt<Tag>::pack2(x[2], x[3]), Elt<Tag>::pack2(x[4], x[5]), Elt<Tag>::pack2(x[6], x[7])};
  }
  static __device__ __forceinline__ Frag zero() { return Frag{0u, 0u, 0u, 0u}; }
  static __device__ __forceinline__ Frag load(const void* p) { return *(const Frag*)p; }
  // a value that is infinite or NaN among 8: its exponent plus one unit carries into the sign's place
  static __device__ __forceinline__ bool odd(const u32x4& x) {
    constexpr uint32_t E = std::is_same_v<Tag, bf16_tag> ? 0x7f807f80u : 0x7c007c00u, U = E & -E & 0xffffu;
    uint32_t any = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) any |= (x[i] & E) + (U << 16 | U);
    return any & 0x80008000u;
  }
  // c + the sum of an operand's values
  static __device__ __forceinline__ float total(const Frag& x, float c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = x[i];  // (a bit cast of the element itself reads element 0)
      if constexpr (std::is_same_v<Tag, bf16_tag>)
        c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0x3f803f80u), c, false);
      else
        c = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), __builtin_bit_cast(f16x2, 0x3c003c00u), c, false);
    }
    return c;
  }
  static __device__ __forceinline__ Frag sign(Frag x, bool neg, bool zero) {  // -x, 0
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = zero ? 0u : neg ? x[i] ^ 0x80008000u : x[i];
    return x;
  }
  static __device__ __forceinline__ Frag finite(Frag x) { return finite16(x); }
  static __device__ __forceinline__ u32x4 finite16(u32x4 x) {  // such values as 0
    constexpr uint32_t E = std::is_same_v<Tag, bf16_tag> ? 0x7f80u : 0x7c00u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] &= ((x[i] & E) == E ? 0u : 0xffffu) | ((x[i] & (E << 16)) == (E << 16) ? 0u : 0xffff0000u);
    return x;
  }
};
template <>
struct SOp<float> {
  using Frag = F8;
  static constexpr int ES = 4;
  static __device__ __forceinline__ f32x16 mma32(const Frag& a, const Frag& b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.a[e], b.a[e], c, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.b[e], b.b[e], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ f32x4 mma16(const Frag& a, const Frag& b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.a[e], b.a[e], c, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.b[e], b.b[e], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag pack(const float (&x)[8]) {
    return Frag{f32x4{x[0], x[1], x[2], x[3]}, f32x4{x[4], x[5], x[6], x[7]}};
  }
  static __device__ __forceinline__ Frag zero() { return Frag{f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}}; }
  static __device__ __forceinline__ Frag load(const void* p) { return Frag{*(const f32x4*)p, *(const f32x4*)((const char*)p + 16)}; }
  static __device__ __forceinline__ bool odd(const u32x4& x) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) any = any || (x[i] & 0x7f800000u) == 0x7f800000u;
    return any;
  }
  static __device__ __forceinline__ float total(const Frag& x, float c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c += x.a[i] + x.b[i];
    return c;
  }
  static __device__ __forceinline__ Frag sign(Frag x, bool neg, bool zero) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x.a[i] = zero ? 0.f : neg ? -x.a[i] : x.a[i];
      x.b[i] = zero ? 0.f : neg ? -x.b[i] : x.b[i];
    }
    return x;
  }
  static __device__ __forceinline__ u32x4 finite16(u32x4 x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (x[i] & 0x7f800000u) == 0x7f800000u ? 0u : x[i];
    return x;
  }
  static __device__ __forceinline__ Frag finite(Frag x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x.a[i] = __builtin_isfinite(x.a[i]) ? x.a[i] : 0.f;
      x.b[i] = __builtin_isfinite(x.b[i]) ? x.b[i] : 0.f;
    }
    return x;
  }
};

// Order of a stretch of code with N products whose operands take R LDS reads each: the
// reads of AHEAD products first, then a product and the reads of a later one in turn.
// (Left to itself the compiler issues each read right before its product and waits.)
template <int N, int AHEAD, int R>
__device__ __forceinline__ void reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * R, 0);  // LDS reads
#pragma unroll
  for (int i = 0; i < N - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix products
    __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}

// A tile of rows of D elements in LDS, packed, 16-byte chunk c of row r at c ^ f(r): row
// reads (16 rows at one chunk) and transposed reads (4 rows at 4 chunks) then touch all
// 64 banks once.
template <class Tag, int D>
struct STile {
  using O = SOp<Tag>;
  static constexpr int RB = D * O::ES, CPR = RB / 16;  // bytes and chunks of a row
  static __device__ __forceinline__ int f(int r) {
    if constexpr (CPR >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    else return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  }
  static __device__ __forceinline__ int at(int r, int c) { return r * RB + ((c ^ f(r)) << 4); }

  // elements 8 k .. 8 k + 7 of row r
  static __device__ __forceinline__ typename O::Frag row(const char* t, int r, int k) {
    if constexpr (O::ES == 2) return *(const u32x4*)(t + at(r, k));
    else return F8{*(const f32x4*)(t + at(r, 2 * k)), *(const f32x4*)(t + at(r, 2 * k + 1))};
  }
  // four rows r .. r + 3 (r % 4 == 0 for the whole 16-lane group) of column c0 + lane % 16
  static __device__ __forceinline__ u32x2 tr4(const char* t, int r, int c0, int lane) {
    const int i = lane & 15, rr = r + (i >> 2), c = (c0 >> 3) + ((i & 3) >> 1);
    using v4s = short __attribute__((ext_vector_type(4)));
    auto p = (__attribute__((address_space(3))) v4s*)(t + at(rr, c) + 8 * (i & 1));
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
  }
  static __device__ __forceinline__ float elem(const char* t, int r, int c) {
    return *(const float*)(t + at(r, c >> 2) + 4 * (c & 3));
  }
  // A operand of a 32x32 product over rows 16 j .. 16 j + 15 of the tile: column 32 mt + l32
  static __device__ __forceinline__ typename O::Frag tr32(const char* t, int j, int mt, int lane) {
    const int hi = lane >> 5, r = 16 * j + 4 * hi;
    if constexpr (O::ES == 2) {
      const int c0 = 32 * mt + 16 * ((lane >> 4) & 1);
      const u32x2 x = tr4(t, r, c0, lane), y = tr4(t, r + 8, c0, lane);
      return u32x4{x[0], x[1], y[0], y[1]};
    } else {
      const int c = 32 * mt + (lane & 31);
      F8 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o.a[e] = elem(t, r + e, c);
        o.b[e] = elem(t, r + 8 + e, c);
      }
      return o;
    }
  }
  // The same in the order of an operand read along its rows (slot e: row 16 j + 8 hi + e)
  static __device__ __forceinline__ typename O::Frag tr32n(const char* t, int j, int mt, int lane) {
    const int hi = lane >> 5, r = 16 * j + 8 * hi;
    if constexpr (O::ES == 2) {
      const int c0 = 32 * mt + 16 * ((lane >> 4) & 1);
      const u32x2 x = tr4(t, r, c0, lane), y = tr4(t, r + 4, c0, lane);
      return u32x4{x[0], x[1], y[0], y[1]};
    } else {
      const int c = 32 * mt + (lane & 31);
      F8 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o.a[e] = elem(t, r + e, c);
        o.b[e] = elem(t, r + 4 + e, c);
      }
      return o;
    }
  }
  // A operand of a 16x16 product over rows 0 .. 31 of the tile: column 16 dt + l16
  static __device__ __forceinline__ typename O::Frag tr16(const char* t, int dt, int lane) {
    const int g = lane >> 4;
    if constexpr (O::ES == 2) {
      const u32x2 x = tr4(t, 4 * g, 16 * dt, lane), y = tr4(t, 16 + 4 * g, 16 * dt, lane);
      return u32x4{x[0], x[1], y[0], y[1]};
    } else {
      const int c = 16 * dt + (lane & 15);
      F8 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o.a[e] = elem(t, 4 * g + e, c);
        o.b[e] = elem(t, 16 + 4 * g + e, c);
      }
      return o;
    }
  }
};

}  // namespace mattn
