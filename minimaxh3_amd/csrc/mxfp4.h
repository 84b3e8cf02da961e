// Blocks of 32 four-bit values under a shared power of two (OCP MX, e2m1 codes and e8m0 scales): the pieces
// that quantizing kernels share.
//
// Codes of a row [K]: K / 2 bytes, two codes a byte, the even element in the low half.  Scales of a matrix
// [M, K]: [ceil(K / 256)][M][8] bytes, exponent + 127 of blocks 8 s .. 8 s + 7 of each row in slab s, so that
// the product reads the scales of one K stage of many rows as whole cache lines.  Bytes of blocks past K hold 127.
#pragma once

#include "common.h"

namespace mxf8 {

constexpr int MX_BLOCK = 32;
constexpr int MX_SLAB = 8;  // blocks per slab: 256 elements of K

__host__ __device__ constexpr int64_t mx_slabs(int64_t K) { return cdiv(K, MX_BLOCK * MX_SLAB); }

// Byte of block `kb` of row m in the scales of an M-row matrix.
__host__ __device__ __forceinline__ int64_t mx_scale_at(int64_t kb, int64_t m, int64_t M) {
  return ((kb / MX_SLAB) * M + m) * MX_SLAB + kb % MX_SLAB;
}

// Scale byte of a block from the bits of its largest |x|: the power that puts it into [3.5, 7), so that the
// largest code is 4 or 6 (above 6, up to 7, it rounds to 6).  The mantissa's carry past 1.75 raises the
// exponent by one.  An infinity or NaN in the block gives 255 (the block reads as NaN), an all-zero one 0.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
  const uint32_t e = (amax_bits + 0x200000u) >> 23;
  return amax_bits >= 0x7f800000u ? 255u : e > 2u ? e - 2u : 0u;
}

// 2^(byte - 127) as fp32 (255: NaN).
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255u ? 0x7fc00000u : byte << 23);
}

// Eight values divided by the scale and rounded to nearest even e2m1 codes, saturating at 6: four bytes.
__device__ __forceinline__ uint32_t mx_codes8(const float (&f)[8], uint32_t byte) {
  const float s = mx_scale_value(byte);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[0], f[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2], f[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[4], f[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[6], f[7], s, 3);
  return w;
}

// A whole block of 16-bit elements in one lane: loaded from any alignment, and quantized to 16 bytes of codes and
// the scale byte, the same as above.  The elements stay packed: their magnitudes are ordered like integers.
struct MxElems {
  typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));
  typedef unsigned short v2us __attribute__((ext_vector_type(2)));
  words4 w[4];
  __device__ __forceinline__ void load(const uint16_t* p) {
#pragma unroll
    for (int q = 0; q < 4; ++q) w[q] = reinterpret_cast<const words4*>(p)[q];
  }
  template <int DT>
  __device__ __forceinline__ uint32_t quantize(v4i& codes) const {
    v2us m = {0, 0};
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(v2us, w[q][i] & 0x7fff7fffu));
    const uint32_t byte = mx_scale_byte(__float_as_uint(Elem<DT>::to_f32(max(m[0], m[1]))));
    const float s = mx_scale_value(byte);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t a = w[q][0], b = w[q][1], c = w[q][2], d = w[q][3];
      uint32_t o = 0;
      if constexpr (DT == MXF8_BF16) {
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(v2bf, a), s, 0);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(v2bf, b), s, 1);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(v2bf, c), s, 2);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(v2bf, d), s, 3);
      } else {
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(v2h, a), s, 0);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(v2h, b), s, 1);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(v2h, c), s, 2);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(v2h, d), s, 3);
      }
      codes[q] = (int)o;
    }
    return byte;
  }
};

// The largest |f| as bits (a NaN is larger than every number) over eight values and the four lanes of a quad,
// which together hold one block.
__device__ __forceinline__ uint32_t mx_block_absmax(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(f[j]) & 0x7fffffffu);
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xb1, 0xf, 0xf, true));  // lane ^ 1
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4e, 0xf, 0xf, true));  // lane ^ 2
  return m;
}

}  // namespace mxf8
