// What the GEMM kernels of the FP8 and the 4-bit linears share: tile configurations, the direct-to-LDS
// operand copies in rows of 128 bytes, fragment reads and output helpers.
#pragma once

#include <type_traits>

#include "common.h"

namespace mxf8 {
constexpr int GEMM_BK = 128;  // bytes of K per stage and row
}

#include "gemm_tiles.h"

namespace mxf8 {

template <int BM_, int BN_, int WM_, int WN_>
struct GemmCfg {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int NW = WM * WN;                        // waves per workgroup
  static constexpr int THREADS = 64 * NW;
  static constexpr int TM = BM / WM / 32;                   // 32x32 tiles per wave along m
  static constexpr int TN = BN / WN / 32;                   // along n
  static constexpr int STAGE = (BM + BN) * GEMM_BK;         // LDS bytes per stage (W tile, then X tile)
  static constexpr int DMA_PER_WAVE = (BM + BN) / 8 / NW;   // 1 KB DMA instructions per wave per stage
  static_assert((BN / 8) % DMA_PER_WAVE == 0, "a wave's DMA rows must lie in one operand");
  static_assert(DMA_PER_WAVE % 2 == 0, "DMA instruction parity must follow the loop index");
};
typedef GemmCfg<256, 256, 4, 2> GemmBig;    // 8 waves, 128 KB LDS, one workgroup per CU
typedef GemmCfg<128, 128, 2, 2> GemmSmall;  // 4 waves, 64 KB LDS, two workgroups per CU

__device__ __forceinline__ v8i lds_frag(const uint8_t* tile, int row, int chunk0) {
  // 32 bytes = logical chunks chunk0, chunk0 + 1 of `row` (swizzled storage)
  const int sw = lds_swz<GEMM_BK>(row);
  const v4i lo = *reinterpret_cast<const v4i*>(tile + row * GEMM_BK + ((chunk0 ^ sw) << 4));
  const v4i hi = *reinterpret_cast<const v4i*>(tile + row * GEMM_BK + (((chunk0 + 1) ^ sw) << 4));
  v8i r;
  r[0] = lo[0]; r[1] = lo[1]; r[2] = lo[2]; r[3] = lo[3];
  r[4] = hi[0]; r[5] = hi[1]; r[6] = hi[2]; r[7] = hi[3];
  return r;
}

__device__ __forceinline__ float gelu_tanh_f32(float z) {
  // 0.5 z (1 + tanh(u)) = z * sigmoid(2u),  u = sqrt(2/pi) (z + 0.044715 z^3)
  const float u2 = z * __builtin_fmaf(0.0713548162726f, z * z, 1.5957691216057308f);  // 2u
  const float e = __builtin_amdgcn_exp2f(-u2 * 1.4426950408889634f);
  return z * __builtin_amdgcn_rcpf(1.0f + e);
}


// fp32 -> bf16 -> fp32 and fp32 pair -> packed bf16 pair, both with the hardware
// round-to-nearest-even conversion (v_cvt_pk_bf16_f32).
__device__ __forceinline__ float bf16r(float f) { return (float)(__bf16)f; }
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{lo, hi}, v2bf));
}
// bf16r of two values with one conversion: the low half moves up, the high half is masked
// (three instructions for two roundings instead of four)
__device__ __forceinline__ void bf16r2(float& a, float& b) {
  const uint32_t w = bf16x2(a, b);
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}

// 16 bytes of an output tile.  Whole tiles leave with non-temporal stores: the kernel never
// reads them back, and streaming the lines out of the L2 early leaves it to the operand panels
// and makes the next kernels' reads wait less on write-backs.  Same process on MI355X: the
// 480p hot-path step 4.758 -> 4.696 ms, and a chained block (each output feeding the next
// kernel) 4.610 -> 4.556 ms; non-temporal attention-output stores, quantizer code stores or
// quantizer loads on top were each slower in the chained block.
__device__ __forceinline__ void store_out16(uint16_t* p, const uint4& v) {
  __builtin_nontemporal_store(v4i{(int)v.x, (int)v.y, (int)v.z, (int)v.w}, reinterpret_cast<v4i*>(p));
}

// Workgroup barrier that waits for this wave's LDS traffic but, unlike __syncthreads(),
// not for its outstanding global->LDS DMA (which must stay in flight across it).
__device__ __forceinline__ void block_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// This wave's share of one stage: DMA_PER_WAVE instructions of 8 rows x 128 bytes each,
// all from one operand (rows past the end of the operand read as zero: buffer range
// check).  Instruction J fills LDS stage rows [8J, 8J + 8): W rows for J < BN/8, X rows
// after.  `lane_off` holds the per-lane source offset for even and odd J.
template <class C>
__device__ __forceinline__ void gemm_dma(__amdgpu_buffer_rsrc_t wrs, __amdgpu_buffer_rsrc_t xrs, uint8_t* stage,
                                         const uint32_t (&lane_off)[2], int K, int wave, int k0) {
  const int J0 = wave * C::DMA_PER_WAVE;
  const bool is_w = J0 < C::BN / 8;
  const __amdgpu_buffer_rsrc_t rs = is_w ? wrs : xrs;
  const int row0 = is_w ? 8 * J0 : 8 * J0 - C::BN;  // first operand row of this wave's share
#pragma unroll
  for (int j = 0; j < C::DMA_PER_WAVE; ++j) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, LDS_PTR(stage + (J0 + j) * 1024), 16, lane_off[j & 1],
                                             (row0 + 8 * j) * K + k0, 0, 0);
  }
}

// Zero the logical 16-byte chunks at or past K of every row of a stage (last, partial
// stage; K % 16 == 0).
template <class C>
__device__ __forceinline__ void zero_tail(uint8_t* stage, int valid_chunks) {
  for (int x = threadIdx.x; x < (C::BM + C::BN) * 8; x += C::THREADS) {
    const int row = x >> 3, c = x & 7;
    if (c >= valid_chunks)
      *reinterpret_cast<v4i*>(stage + row * GEMM_BK + ((c ^ lds_swz<GEMM_BK>(row)) << 4)) = v4i{0, 0, 0, 0};
  }
}

}  // namespace mxf8
