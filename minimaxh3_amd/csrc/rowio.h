// Eight elements of a row at a time, as fp32: loads and stores of the element-wise kernels (rotary.hip,
// block_norm.hip, mxfp4.hip).  gfx950 takes a 16-byte access at any element's address, so rows of odd
// lengths and views that start anywhere go the same way as aligned ones.
#pragma once

#include "common.h"

namespace mxf8 {

struct __attribute__((packed, aligned(2))) Words4 {
  uint32_t w[4];
};
struct __attribute__((packed, aligned(4))) Floats4 {
  float f[4];
};

template <int DT>
struct Raw8 {
  uint32_t w[4];
  __device__ __forceinline__ void load(const void* base, int64_t i) {
    const Words4 v = *reinterpret_cast<const Words4*>(static_cast<const uint16_t*>(base) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = v.w[j];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = 0;
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[2 * j] = Elem<DT>::lo(w[j]), f[2 * j + 1] = Elem<DT>::hi(w[j]);
  }
  // rounds to nearest even
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = cvt_pk_16<DT>(f[2 * j], f[2 * j + 1]);
  }
  __device__ __forceinline__ void store(void* base, int64_t i) const {
    *reinterpret_cast<Words4*>(static_cast<uint16_t*>(base) + i) = Words4{{w[0], w[1], w[2], w[3]}};
  }
};

template <>
struct Raw8<MXF8_F32> {
  float w[8];
  __device__ __forceinline__ void load(const void* base, int64_t i) {
    const float* p = static_cast<const float*>(base) + i;
    const Floats4 a = *reinterpret_cast<const Floats4*>(p), b = *reinterpret_cast<const Floats4*>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = a.f[j], w[j + 4] = b.f[j];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = 0.0f;
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = w[j];
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = f[j];
  }
  __device__ __forceinline__ void store(void* base, int64_t i) const {
    float* p = static_cast<float*>(base) + i;
    *reinterpret_cast<Floats4*>(p) = Floats4{{w[0], w[1], w[2], w[3]}};
    *reinterpret_cast<Floats4*>(p + 4) = Floats4{{w[4], w[5], w[6], w[7]}};
  }
};

// One element.
template <int DT>
__device__ __forceinline__ float load1(const void* base, int64_t i) {
  return Elem<DT>::to_f32(static_cast<const typename Elem<DT>::T*>(base)[i]);
}
// f rounded to the type.
template <int DT>
__device__ __forceinline__ float round1(float f) {
  if constexpr (DT == MXF8_F32)
    return f;
  else
    return Elem<DT>::lo(cvt_pk_16<DT>(f, f));
}
template <int DT>
__device__ __forceinline__ void store1(void* base, int64_t i, float f) {
  if constexpr (DT == MXF8_F32)
    static_cast<float*>(base)[i] = f;
  else
    static_cast<uint16_t*>(base)[i] = (uint16_t)cvt_pk_16<DT>(f, f);
}

}  // namespace mxf8
