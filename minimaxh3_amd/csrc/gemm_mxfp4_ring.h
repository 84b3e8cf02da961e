// The 4-bit linear for few tokens: the same products as gemm_mxfp4_kernel (gemm_mxfp4.hip), which keeps two
// stages of copies in flight and needs hundreds of output tiles to fill the chip.
//
// gemm_mxfp4_ring_kernel: one small tile per workgroup, stages of K in a deep LDS ring, as gemm_ring.h has it
// for FP8.  What bounds it is the chain of stages: a stage's copies are issued NS - 1 stages ahead, and its
// fragments are read from LDS while the previous stage's products run.  513 x 3072 x 3072 8.9-10.7 us, a stage of a 128 x 64
// tile about 1050 cycles, of which LDS serves reads and copies for 700.  Rings twice as deep (9.4), two or three stages
// to a barrier (10.4, 9.6) and waves of 64 x 32 outputs (10.9) were slower.
//
// gemm_mxfp4_rows_kernel: products too small to give every compute unit a tile.  Little is shared there, so no
// operand goes through LDS and no wave waits for another: each of a workgroup's waves streams the weights of
// 16 or 32 channels over its own slabs of K straight into fragments, and the partial sums meet in LDS at the end.
// 1 x 9216 x 3072, activations quantized here, 6.1 us: 15.3 MB at 2.5 TB/s, the latency of two rounds of loads and of
// the launch (1.9 us).
#pragma once

#include "gemm_common.h"
#include "mxfp4.h"

namespace mxf8 {

__device__ __forceinline__ v8i mx_wide(const v4i& v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

// One instruction on block 4 g + T of the stage: 16 bytes of each operand per lane, byte T of the scale dwords.
template <int T>
__device__ __forceinline__ v16f mx_mma(const v4i& a, const v4i& b, const v16f& c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_wide(a), mx_wide(b), c, 4, 4, T, (int)sa, T, (int)sb);
}

// 16 bytes: logical chunk `chunk` of `row` (swizzled storage).
__device__ __forceinline__ v4i mx_frag(const uint8_t* tile, int row, int chunk) {
  return *reinterpret_cast<const v4i*>(tile + row * GEMM_BK + ((chunk ^ lds_swz<GEMM_BK>(row)) << 4));
}

// GELU-tanh, z sigmoid(2 u) with u = sqrt(2 / pi) (z + 0.044715 z^3), as z / (1 + 2^t): t = -2 u log2(e), whose two
// coefficients hold all constants (at 12288 channels the activation is an eighth of the kernel's cycles).
__device__ __forceinline__ float mx_gelu(float z) {
  const float t = z * __builtin_fmaf(-0.10294324f, z * z, -2.3022082f);
  return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t));
}

template <int ACT>
__device__ __forceinline__ uint2 mx_out_quad(const v4f& x, const v4f& b) {
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = x[e] + b[e];
    if constexpr (ACT == MXF8_ACT_GELU_TANH) v[e] = mx_gelu(v[e]);
  }
  return make_uint2(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]));
}

// The first n of eight outputs (none for n <= 0), at any alignment: one store if all are there.  STREAM: past the
// caches (store_out16's reasons hold for large outputs).
typedef uint32_t mx_words4 __attribute__((ext_vector_type(4), aligned(2)));
template <bool STREAM>
__device__ __forceinline__ void mx_store8(uint16_t* dst, const uint4& v, int n) {
  if (n >= 8) {
    const mx_words4 w = {v.x, v.y, v.z, v.w};
    if constexpr (STREAM)
      __builtin_nontemporal_store(w, reinterpret_cast<mx_words4*>(dst));
    else
      *reinterpret_cast<mx_words4*>(dst) = w;
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) dst[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
  }
}

// A wave's share of the copies of a stage's scales, BN rows of W, then BM rows of X, from the tile's first rows of the
// slab: 256-byte instructions of 32 rows, two dwords a row.  Rows past the operand's end (wrows, xrows of them are
// there) read as zeros (2^-127, with zero codes).  Every wave issues as many instructions (some copy rows again), so
// that one count of instructions in flight holds for all.
template <class C>
__device__ __forceinline__ void mx_copy_scales(const uint8_t* w, const uint8_t* x, int wrows, int xrows, uint8_t* dst,
                                               int wave, int lane) {
  constexpr int ALL = (C::BM + C::BN) / 32;
#pragma unroll
  for (int j = 0; j < (ALL + C::NW - 1) / C::NW; ++j) {
    // (whole rounds of the waves over each operand: known here which)
    constexpr bool whole = C::BN / 32 % C::NW == 0 && ALL % C::NW == 0;
    const int J = whole ? wave + j * C::NW : (wave + j * C::NW) % ALL;
    const bool is_w = whole ? j * C::NW < C::BN / 32 : J < C::BN / 32;
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void*)(is_w ? w : x), 0, (is_w ? wrows : xrows) * MX_SLAB, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, LDS_PTR(dst + J * 256), 4, lane * 4,
                                             (is_w ? 32 * J : 32 * J - C::BN) * MX_SLAB, 0, 0);
  }
}

template <int BM_, int BN_, int WM_, int WN_, int NS_>
struct MxRing {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NS = NS_;
  static constexpr int NW = WM * WN, THREADS = 64 * NW;
  static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
  static constexpr int CODES = (BM + BN) * GEMM_BK;          // LDS bytes of a stage: W rows, then X rows,
  static constexpr int STAGE = CODES + (BM + BN) * MX_SLAB;  // and their scales in the same order
  static constexpr int DMA_CODES = (BM + BN) / 8 / NW;       // 1 KB instructions per wave and stage
  static constexpr int DMA_SCALES = ((BM + BN) / 32 + NW - 1) / NW;      // and of mx_copy_scales
  static constexpr int PER_STAGE = DMA_CODES + DMA_SCALES;
  static constexpr int OUT_PITCH = BN * 2 + 16;
  static_assert((BM + BN) / 8 % NW == 0 && BN % 32 == 0 && BM % 32 == 0, "DMA shares");
  static_assert(NS * STAGE + BN * 4 <= 160 * 1024 && BM * OUT_PITCH <= NS * STAGE, "LDS");
  static_assert(NS >= 3 && (NS - 1) * PER_STAGE < 64, "vmcnt counts the copies of NS - 1 stages");

  // This wave's share of a stage's codes, as gemm_dma, whichever operand each instruction's 8 rows belong to.
  static __device__ __forceinline__ void copy_codes(__amdgpu_buffer_rsrc_t wrs, __amdgpu_buffer_rsrc_t xrs,
                                                    uint8_t* stage, const uint32_t (&lane_off)[2], int Kb, int wave,
                                                    int k0) {
#pragma unroll
    for (int j = 0; j < DMA_CODES; ++j) {
      const int J = wave * DMA_CODES + j;
      const bool is_w = J < BN / 8;
      const __amdgpu_buffer_rsrc_t rs = is_w ? wrs : xrs;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, LDS_PTR(stage + J * 1024), 16, lane_off[J & 1],
                                               (is_w ? 8 * J : 8 * J - BN) * Kb + k0, 0, 0);
    }
  }
};

template <class C, int ACT, bool KTAIL>
__global__ __launch_bounds__(C::THREADS) void gemm_mxfp4_ring_kernel(const uint8_t* __restrict__ a4, const uint8_t* __restrict__ w4,
                                                                     const uint8_t* __restrict__ sa,
                                                                     const uint8_t* __restrict__ sw,
                                                                     const uint16_t* __restrict__ bias,
                                                                     uint16_t* __restrict__ out, int M, int N, int Kb,
                                                                     int64_t ld_out, int tiles_m, int tiles_n) {
  constexpr int TM = C::TM, TN = C::TN, NS = C::NS;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[NS * C::STAGE];
  __shared__ __attribute__((aligned(16))) float ep_b[C::BN];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wn = wave / C::WM, wm = wave % C::WM;
  const int wrow0 = wn * (C::BN / C::WN), xrow0 = wm * (C::BM / C::WM);
  const int nk = (Kb + GEMM_BK - 1) / GEMM_BK;
  const int r = lane & 31, g = lane >> 5;
  int tm, tn;
  tile_coords(blockIdx.x, tiles_m, tiles_n, RING_GROUP_M, tm, tn);
  const int m0 = tm * C::BM, n0 = tn * C::BN;
  uint32_t lane_off[2];
#pragma unroll
  for (int par = 0; par < 2; ++par)
    lane_off[par] = (uint32_t)((lane >> 3) * Kb) +
                    (uint32_t)(((lane & 7) ^ lds_swz<GEMM_BK>(8 * par + (lane >> 3))) << 4);
  auto rsrc = [&](const uint8_t* base, int row0, int rows, int span) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)(base + (int64_t)row0 * Kb), 0, min(rows - row0, span) * Kb,
                                             0x00020000);
  };
  const __amdgpu_buffer_rsrc_t wrs = rsrc(w4, n0, N, C::BN), xrs = rsrc(a4, m0, M, C::BM);
  auto dma = [&](uint8_t* stage, int ks) {
    C::copy_codes(wrs, xrs, stage, lane_off, Kb, wave, ks * GEMM_BK);
    mx_copy_scales<C>(sw + ((int64_t)ks * N + n0) * MX_SLAB, sa + ((int64_t)ks * M + m0) * MX_SLAB, min(N - n0, C::BN),
                   min(M - m0, C::BM), stage + C::CODES, wave, lane);
  };
  // the bias, read before the copies that the waits below count, handed over through LDS
  constexpr int NEP = (C::BN + C::THREADS - 1) / C::THREADS;
  uint16_t ep_v[NEP];
#pragma unroll
  for (int e = 0; e < NEP; ++e)
    ep_v[e] = *(bias ? bias + min(n0 + (int)threadIdx.x + e * C::THREADS, N - 1) : reinterpret_cast<const uint16_t*>(sw));
#pragma unroll
  for (int s = 0; s < NS; ++s)
    if (s < nk) dma(smem + s * C::STAGE, s);
#pragma unroll
  for (int e = 0; e < NEP; ++e) {
    const int i = threadIdx.x + e * C::THREADS;
    if (i < C::BN) ep_b[i] = bias ? bf16_bits_to_f32(ep_v[e]) : 0.0f;
  }

  v16f acc[TN][TM];
#pragma unroll
  for (int a = 0; a < TN; ++a)
#pragma unroll
    for (int b = 0; b < TM; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.0f;

  // One stage's fragments: block 4 g + t of each of this lane's rows for step t, and the rows' scale dwords.
  struct Frags {
    v4i a[4][TN], b[4][TM];
    uint32_t sa[TN], sb[TM];
  };
  auto read = [&](const uint8_t* st, Frags& f) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int a = 0; a < TN; ++a) f.a[t][a] = mx_frag(st, wrow0 + 32 * a + r, 4 * g + t);
#pragma unroll
      for (int b = 0; b < TM; ++b) f.b[t][b] = mx_frag(st + C::BN * GEMM_BK, xrow0 + 32 * b + r, 4 * g + t);
    }
#pragma unroll
    for (int a = 0; a < TN; ++a)
      f.sa[a] = *reinterpret_cast<const uint32_t*>(st + C::CODES + (wrow0 + 32 * a + r) * MX_SLAB + 4 * g);
#pragma unroll
    for (int b = 0; b < TM; ++b)
      f.sb[b] = *reinterpret_cast<const uint32_t*>(st + C::CODES + (C::BN + xrow0 + 32 * b + r) * MX_SLAB + 4 * g);
  };
  // The last stage's blocks past K: zero codes, and scales of 1 in the place of bytes that may hold anything.
  auto mend = [&](uint8_t* st) {
    const int valid = (Kb % GEMM_BK) >> 4;
    zero_tail<C>(st, valid);
    for (int x = threadIdx.x; x < (C::BM + C::BN) * MX_SLAB; x += C::THREADS)
      if (x % MX_SLAB >= valid) st[C::CODES + x] = 127;
  };
  auto landed = [&](int ks, auto in_flight) {
    if (ks + decltype(in_flight)::value >= nk)
      wait_vm0();
    else
      wait_vm<decltype(in_flight)::value * C::PER_STAGE>();
    block_barrier();
    if (KTAIL && ks == nk - 1) {
      mend(smem + (ks % NS) * C::STAGE);
      block_barrier();
    }
  };
  auto products = [&](const Frags& f) {
#pragma unroll
    for (int a = 0; a < TN; ++a)
#pragma unroll
      for (int b = 0; b < TM; ++b) {
        acc[a][b] = mx_mma<0>(f.a[0][a], f.b[0][b], acc[a][b], f.sa[a], f.sb[b]);
        acc[a][b] = mx_mma<1>(f.a[1][a], f.b[1][b], acc[a][b], f.sa[a], f.sb[b]);
        acc[a][b] = mx_mma<2>(f.a[2][a], f.b[2][b], acc[a][b], f.sa[a], f.sb[b]);
        acc[a][b] = mx_mma<3>(f.a[3][a], f.b[3][b], acc[a][b], f.sa[a], f.sb[b]);
      }
  };
  int slot = 0;  // ks % NS
  Frags f0, f1;
  landed(0, std::integral_constant<int, NS - 1>{});
  read(smem, f0);
  auto stage = [&](int ks, const Frags& cur, Frags& nxt) {
    const int next = slot + 1 == NS ? 0 : slot + 1;
    if (ks + 1 < nk) {
      landed(ks + 1, std::integral_constant<int, NS - 2>{});
      if (ks + NS < nk) dma(smem + slot * C::STAGE, ks + NS);
      read(smem + next * C::STAGE, nxt);
    }
    slot = next;
    products(cur);
  };
  for (int ks = 0; ks < nk; ks += 2) {
    stage(ks, f0, f1);
    if (ks + 1 < nk) stage(ks + 1, f1, f0);
  }

  // ---- epilogue: acc[a][b] register i is channel n0 + wrow0 + 32 a + 8 (i / 4) + 4 g + i % 4 of token
  // m0 + xrow0 + 32 b + r
  block_barrier();  // every wave has read its last fragments: the ring takes the output tile
#pragma unroll
  for (int a = 0; a < TN; ++a)
#pragma unroll
    for (int b = 0; b < TM; ++b)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int nl = wrow0 + 32 * a + 8 * q + 4 * g;
        *reinterpret_cast<uint2*>(smem + (xrow0 + 32 * b + r) * C::OUT_PITCH + 2 * nl) =
            mx_out_quad<ACT>(v4f{acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]},
                             *reinterpret_cast<const v4f*>(ep_b + nl));
      }
  block_barrier();
  constexpr int CPR = C::BN / 8;  // 16-byte chunks per staged row
  for (int x = threadIdx.x; x < C::BM * CPR; x += C::THREADS) {
    const int row = x / CPR, c = x % CPR, m = m0 + row, n = n0 + 8 * c;
    if (m >= M || n >= N) continue;
    const uint4 v = *reinterpret_cast<const uint4*>(smem + row * C::OUT_PITCH + 16 * c);
    mx_store8<false>(out + (int64_t)m * ld_out + n, v, N - n);
  }
}

// 16 TN channels x 16 TM tokens per workgroup of NW waves.  A unit is one slab of K (256 elements, 128 bytes of a
// row): lane group g = lane / 16 of the 16 x 16 x 128 instruction takes blocks 2 g and 2 g + 1 of its row, one
// per instruction, 32 bytes and two scale bytes.  Wave w takes units w, w + NW, ..., up to four in flight.
//
// XT: the activations are codes and scales (MX_CODES), or 16-bit elements of that type, row stride ldx, which each
// workgroup quantizes for itself into LDS, where that costs less than a launch of its own.
constexpr int MX_CODES = -1;

template <int T>
__device__ __forceinline__ v4f mx_mma16(const v4i& a, const v4i& b, const v4f& c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_wide(a), mx_wide(b), c, 4, 4, T, (int)sa, T, (int)sb);
}

// LDS bytes of one such row of nk slabs, and 16 more (rows of a multiple of 128 bytes would all start in one bank).
__host__ __device__ constexpr int mx_row_pitch(int nk) { return nk * GEMM_BK + ((nk * MX_SLAB + 15) & ~15) + 16; }

template <int TM, int TN, int NW, int ACT, bool KTAIL, int XT>
__global__ __launch_bounds__(64 * NW) void gemm_mxfp4_rows_kernel(const void* __restrict__ x, int64_t ldx,
                                                                  const uint8_t* __restrict__ sa,
                                                                  const uint8_t* __restrict__ w4,
                                                                  const uint8_t* __restrict__ sw,
                                                                  const uint16_t* __restrict__ bias,
                                                                  uint16_t* __restrict__ out, int M, int N, int Kb,
                                                                  int64_t ld_out) {
  __shared__ __attribute__((aligned(16))) v4f part[NW][TN * TM][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16 * TN, m0 = blockIdx.y * 16 * TM;
  const int nk = (Kb + GEMM_BK - 1) / GEMM_BK;
  extern __shared__ __attribute__((aligned(16))) uint8_t xq[];  // activations quantized here: a row's codes, then its scales
  const int pitch = mx_row_pitch(nk);
  // rows past the end are the last row again (not stored)
  const uint8_t *wp[TN], *swp[TN], *xp[TM], *sxp[TM];
#pragma unroll
  for (int a = 0; a < TN; ++a) {
    const int row = min(n0 + 16 * a + r, N - 1);
    wp[a] = w4 + (int64_t)row * Kb + 32 * g;
    swp[a] = sw + (int64_t)row * MX_SLAB + 2 * g;
  }
#pragma unroll
  for (int b = 0; b < TM; ++b) {
    const int row = min(m0 + 16 * b + r, M - 1);
    if constexpr (XT == MX_CODES) {
      xp[b] = static_cast<const uint8_t*>(x) + (int64_t)row * Kb + 32 * g;
      sxp[b] = sa + (int64_t)row * MX_SLAB + 2 * g;
    } else {
      xp[b] = xq + row * pitch + 32 * g;
      sxp[b] = xq + row * pitch + nk * GEMM_BK + 2 * g;
    }
  }
  struct Operand {
    v4i c[2];
    uint32_t s;
  };
  // blocks 2 g and 2 g + 1 of slab ks; those past K, in the last one, are zero codes under a scale of 1
  const v4i none = {0, 0, 0, 0};
  auto load = [&](const uint8_t* p, const uint8_t* s, int ks, Operand& o) {
    const int n = KTAIL && ks + 1 == nk ? (Kb >> 4) - 8 * ks - 2 * g : 2;
    if (!KTAIL || ks + 1 < nk || n >= 2) {
      o.c[0] = *reinterpret_cast<const v4i*>(p);
      o.c[1] = *reinterpret_cast<const v4i*>(p + 16);
      o.s = *reinterpret_cast<const uint16_t*>(s);
    } else {
      o.c[0] = n == 1 ? *reinterpret_cast<const v4i*>(p) : none;
      o.c[1] = none;
      o.s = 0x7f00u | (n == 1 ? s[0] : 127u);
    }
  };
  struct Unit {
    Operand w[TN], x[TM];
  };
  auto load_w = [&](int ks, Unit& u) {
#pragma unroll
    for (int a = 0; a < TN; ++a)
      load(wp[a] + (int64_t)ks * GEMM_BK, swp[a] + (int64_t)ks * N * MX_SLAB, ks, u.w[a]);
  };
  auto load_x = [&](int ks, Unit& u) {
#pragma unroll
    for (int b = 0; b < TM; ++b) {
      if constexpr (XT == MX_CODES) {
        load(xp[b] + (int64_t)ks * GEMM_BK, sxp[b] + (int64_t)ks * M * MX_SLAB, ks, u.x[b]);
      } else {
        u.x[b].c[0] = *reinterpret_cast<const v4i*>(xp[b] + ks * GEMM_BK);
        u.x[b].c[1] = *reinterpret_cast<const v4i*>(xp[b] + ks * GEMM_BK + 16);
        u.x[b].s = *reinterpret_cast<const uint16_t*>(sxp[b] + ks * MX_SLAB);
      }
    }
  };
  v4f acc[TN][TM];
#pragma unroll
  for (int a = 0; a < TN; ++a)
#pragma unroll
    for (int b = 0; b < TM; ++b) acc[a][b] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  auto products = [&](const Unit& u) {
#pragma unroll
    for (int a = 0; a < TN; ++a)
#pragma unroll
      for (int b = 0; b < TM; ++b) {
        acc[a][b] = mx_mma16<0>(u.w[a].c[0], u.x[b].c[0], acc[a][b], u.w[a].s, u.x[b].s);
        acc[a][b] = mx_mma16<1>(u.w[a].c[1], u.x[b].c[1], acc[a][b], u.w[a].s, u.x[b].s);
      }
  };
  constexpr int DEPTH = NW == 16 ? 2 : 4;
  Unit u[DEPTH];
  auto load_ahead = [&] {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
      if (wave + d * NW < nk) load_w(wave + d * NW, u[d]);
  };
  if constexpr (XT == MX_CODES) {
    load_ahead();
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
      if (wave + d * NW < nk) load_x(wave + d * NW, u[d]);
  } else {
    // A block per thread at a time, the first ones loaded before the weights: loads return in order, and what
    // quantizing takes passes while the weights come.
    constexpr int THREADS = 64 * NW, FIRST = 2;
    const int per_row = nk * MX_SLAB, blocks = M * per_row;
    MxElems e[FIRST];
    auto source = [&](int i, int& row, int& kb) {
      row = i / per_row;
      kb = i - row * per_row;
      return i < blocks && kb < Kb >> 4;
    };
    auto fetch = [&](int i, MxElems& to) {
      int row, kb;
      if (source(i, row, kb)) to.load(static_cast<const uint16_t*>(x) + row * ldx + kb * MX_BLOCK);
    };
    auto put = [&](int i, const MxElems& from) {
      int row, kb;
      const bool is = source(i, row, kb);
      v4i c = none;
      uint32_t byte = 127;  // blocks past K: zeros under a scale of 1
      if (is) byte = from.template quantize<XT>(c);
      if (i < blocks) {
        *reinterpret_cast<v4i*>(xq + row * pitch + kb * 16) = c;
        xq[row * pitch + nk * GEMM_BK + kb] = (uint8_t)byte;
      }
    };
#pragma unroll
    for (int j = 0; j < FIRST; ++j) fetch(threadIdx.x + j * THREADS, e[j]);
    __builtin_amdgcn_sched_barrier(0);
    load_ahead();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < FIRST; ++j) put(threadIdx.x + j * THREADS, e[j]);
    for (int i = threadIdx.x + FIRST * THREADS; i < blocks; i += THREADS) {
      fetch(i, e[0]);
      put(i, e[0]);
    }
    block_barrier();
  }
  for (int ks = wave; ks < nk; ks += DEPTH * NW) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (ks + d * NW < nk) {
        if (XT != MX_CODES) load_x(ks + d * NW, u[d]);
        products(u[d]);
        if (ks + (d + DEPTH) * NW < nk) {
          load_w(ks + (d + DEPTH) * NW, u[d]);
          if (XT == MX_CODES) load_x(ks + (d + DEPTH) * NW, u[d]);
        }
      }
    }
  }
#pragma unroll
  for (int a = 0; a < TN; ++a)
#pragma unroll
    for (int b = 0; b < TM; ++b) part[wave][a * TM + b][lane] = acc[a][b];
  __syncthreads();
  // part[.][a TM + b][lane]: channels n0 + 16 a + 4 g .. + 3 of token m0 + 16 b + r; thread t sums entry t over the waves
  for (int e = threadIdx.x; e < TN * TM * 64; e += 64 * NW) {
    const int t = e >> 6, l = e & 63, m = m0 + 16 * (t % TM) + (l & 15), n = n0 + 16 * (t / TM) + 4 * (l >> 4);
    if (m >= M || n >= N) continue;
    v4f s = part[0][t][l];
#pragma unroll
    for (int w = 1; w < NW; ++w) s += part[w][t][l];
    v4f bq = {0.0f, 0.0f, 0.0f, 0.0f};
    if (bias) {
#pragma unroll
      for (int i = 0; i < 4; ++i) bq[i] = bf16_bits_to_f32(bias[min(n + i, N - 1)]);
    }
    const uint2 o = mx_out_quad<ACT>(s, bq);
    uint16_t* dst = out + (int64_t)m * ld_out + n;
    typedef uint32_t words2 __attribute__((ext_vector_type(2), aligned(2)));
    if (n + 4 <= N) {
      *reinterpret_cast<words2*>(dst) = words2{o.x, o.y};
    } else {
      const uint32_t w[2] = {o.x, o.y};
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (n + i < N) dst[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
  }
}

}  // namespace mxf8
