// Eight elements of a row at a time, as fp32: loads and stores of the element-wise kernels (rotary.hip,
// block_norm.hip, mxfp4.hip).  gfx950 takes a 16-byte access at any element's address, so rows of odd
// lengths and views that start anywhere go the same way as aligned ones.
#pragma once

#include "common.h"

namespace mxf8 {

typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));
typedef float floats4 __attribute__((ext_vector_type(4), aligned(4)));
// (global memory by name: the compiler does not see it through a choice of two bases)
typedef const __attribute__((address_space(1))) words4* gwords4;
typedef const __attribute__((address_space(1))) floats4* gfloats4;
typedef const __attribute__((address_space(1))) uint8_t* gbytes;

template <int DT>
struct Raw8 {
  uint32_t w[4];
  __device__ __forceinline__ void load(const void* base, int64_t i) { load_at((gbytes)base + i * 2); }
  // non-temporal: for operands that are read once and too large for the caches
  __device__ __forceinline__ void load_stream(const void* base, int64_t i) {
    const words4 v = __builtin_nontemporal_load((gwords4)((gbytes)base + i * 2));
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = v[j];
  }
  // `off`: bytes from a base that is the same for the whole wave
  __device__ __forceinline__ void load_off(const void* base, uint32_t off) { load_at((gbytes)base + off); }
  __device__ __forceinline__ void load_at(gbytes p) {
    const words4 v = *(gwords4)p;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = v[j];
  }
  // elements [0, n) of the eight, n < 8, one by one; the others are 0 / stay as they are
  __device__ __forceinline__ void load_part(const void* base, int64_t i, int n) {
    const uint16_t* p = static_cast<const uint16_t*>(base) + i;
    fill(0.0f);
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < n) w[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
  }
  __device__ __forceinline__ void store_part(void* base, int64_t i, int n) const {
    uint16_t* p = static_cast<uint16_t*>(base) + i;
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < n) p[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
  }
  __device__ __forceinline__ void fill(float f) {
    const uint32_t v = cvt_pk_16<DT>(f, f);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = v;
  }
  __device__ __forceinline__ void zero() { fill(0.0f); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[2 * j] = Elem<DT>::lo(w[j]), f[2 * j + 1] = Elem<DT>::hi(w[j]);
  }
  // The compiler takes the value for another from here on, and unpacks it again for its next use where it would
  // keep the unpacked eight.
  __device__ __forceinline__ void hide() {
#pragma unroll
    for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(w[j]));
  }
  // lane `from`'s eight
  __device__ __forceinline__ void from_lane(int from) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __shfl(w[j], from, 64);
  }
  // rounds to nearest even
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = cvt_pk_16<DT>(f[2 * j], f[2 * j + 1]);
  }
  // non-temporal: for results that the caches would not hold until they are read
  __device__ __forceinline__ void stream(void* base, int64_t i) const {
    stream_off(static_cast<uint16_t*>(base) + i, 0);
  }
  __device__ __forceinline__ void stream_off(void* base, uint32_t off) const {
    __builtin_nontemporal_store(words4{w[0], w[1], w[2], w[3]}, reinterpret_cast<words4*>(static_cast<char*>(base) + off));
  }
};

template <>
struct Raw8<MXF8_F32> {
  float w[8];
  __device__ __forceinline__ void load(const void* base, int64_t i) { load_at((gbytes)base + i * 4); }
  __device__ __forceinline__ void load_stream(const void* base, int64_t i) {
    const floats4 a = __builtin_nontemporal_load((gfloats4)((gbytes)base + i * 4));
    const floats4 b = __builtin_nontemporal_load((gfloats4)((gbytes)base + i * 4 + 16));
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = a[j], w[j + 4] = b[j];
  }
  __device__ __forceinline__ void load_off(const void* base, uint32_t off) { load_at((gbytes)base + off); }
  __device__ __forceinline__ void load_at(gbytes p) {
    const floats4 a = *(gfloats4)p, b = *(gfloats4)(p + 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = a[j], w[j + 4] = b[j];
  }
  __device__ __forceinline__ void load_part(const void* base, int64_t i, int n) {
    const float* p = static_cast<const float*>(base) + i;
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = j < n ? p[j] : 0.0f;
  }
  __device__ __forceinline__ void store_part(void* base, int64_t i, int n) const {
    float* p = static_cast<float*>(base) + i;
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < n) p[j] = w[j];
  }
  __device__ __forceinline__ void fill(float f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = f;
  }
  __device__ __forceinline__ void zero() { fill(0.0f); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = w[j];
  }
  __device__ __forceinline__ void hide() {}
  __device__ __forceinline__ void from_lane(int from) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = __shfl(w[j], from, 64);
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = f[j];
  }
  __device__ __forceinline__ void stream(void* base, int64_t i) const { stream_off(static_cast<float*>(base) + i, 0); }
  __device__ __forceinline__ void stream_off(void* base, uint32_t off) const {
    float* p = reinterpret_cast<float*>(static_cast<char*>(base) + off);
    __builtin_nontemporal_store(floats4{w[0], w[1], w[2], w[3]}, reinterpret_cast<floats4*>(p));
    __builtin_nontemporal_store(floats4{w[4], w[5], w[6], w[7]}, reinterpret_cast<floats4*>(p + 4));
  }
};

// f over the L (8 to 64, a power of two) neighbouring lanes that hold a row or a head, in every one of them: steps within
// rows of 16 lanes and two swaps of rows, all on the vector unit (a shuffle goes through LDS, with some 100 cycles
// a step on a row's critical path).
template <int L, class F>
__device__ __forceinline__ float lanes_reduce(float v, F f) {
  static_assert(L == 8 || L == 16 || L == 32 || L == 64, "lanes of a group");
  v = f(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xb1, 0xf, 0xf, true)));
  v = f(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4e, 0xf, 0xf, true)));
  v = f(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x141, 0xf, 0xf, true)));
  if constexpr (L >= 16)
    v = f(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x140, 0xf, 0xf, true)));
  if constexpr (L >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  if constexpr (L >= 64) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
  return lanes_reduce<L>(v, [](float a, float b) { return a + b; });
}
template <int L>
__device__ __forceinline__ float lanes_max(float v) {
  return lanes_reduce<L>(v, [](float a, float b) { return fmaxf(a, b); });
}

// One element, rounded.
template <int DT>
__device__ __forceinline__ void store1(void* base, int64_t i, float f) {
  if constexpr (DT == MXF8_F32)
    static_cast<float*>(base)[i] = f;
  else
    static_cast<uint16_t*>(base)[i] = (uint16_t)cvt_pk_16<DT>(f, f);
}

}  // namespace mxf8
