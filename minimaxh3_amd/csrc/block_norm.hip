// What stands between two branches of a DiT block, in one pass over its rows:
//
//   u = branch, or branch / sqrt(mean(branch^2) + eps) * branch_weight         (the norm after a branch)
//   r = residual_scale * x + gate * u                                          (the residual stream, stored)
//   n = (r - mean(r)) / sqrt(var(r) + eps)  or  r / sqrt(mean(r^2) + eps)      (the norm before the next branch)
//   y = n * weight * (1 + scale) + shift
//
// and y leaves as it is, or as the e4m3 codes with a row scale that quant_rows gives for it (the FP8 linear's
// input), or as mxfp4_quant's 4-bit blocks (the 4-bit linear's input).  gate, shift and scale are one row per
// span of tokens (a batch item, a frame).  Sums and statistics are fp32 over the unrounded r, held in registers;
// r and y are rounded once each, and codes are those of the rounded y, as if it had been stored and read back.
#include "mxfp4.h"
#include "rowio.h"

namespace mxf8 {

struct BlockNormArgs {
  const void *x, *branch, *gate, *shift, *scale, *branch_weight, *weight;
  void *r, *y;
  uint8_t *codes, *mx_scales;
  float* row_scale;
  int64_t x_b, x_s, br_b, br_s;                    // batch and token strides
  int64_t g_b, g_s, sh_b, sh_s, sc_b, sc_s;        // batch and span strides of the modulation rows
  int S, M;
  int span;  // tokens per modulation row
  int C, layer;
  float eps, residual_scale;
};

// Sum over the NT threads that hold a row, in every one of them.  PARTS: one wave holds what that many waves would
// (its chunk c is the one that wave c % 4 of four has), and adds each one's part as that wave would, then the
// parts in the waves' order: a row's sums do not depend on whether one wave or four hold it (20280 x 3072 in bf16 87.0 us,
// with one sum over the wave 87.6; 10166 x 2730 47.0 / 46.6).
template <int NT, int PARTS>
__device__ __forceinline__ float row_sum(const float (&part)[PARTS], float* red) {
  static_assert(PARTS == 1 || NT == 64, "parts of a wave's row");
  float v = lanes_sum<(NT < 64 ? NT : 64)>(part[0]);
#pragma unroll
  for (int i = 1; i < PARTS; ++i) v += lanes_sum<64>(part[i]);
  if constexpr (NT > 64) {
    const int w = threadIdx.x >> 6;
    __syncthreads();  // the last reduction's values have been read
    if ((threadIdx.x & 63) == 0) red[w] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) v += red[i];
  }
  return v;
}

template <int NT>
__device__ __forceinline__ float row_max(float v, float* red) {
  v = lanes_max<(NT < 64 ? NT : 64)>(v);
  if constexpr (NT > 64) {
    const int w = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[w] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) v = fmaxf(v, red[i]);
  }
  return v;
}

// What stands in for an absent gate, weight (1) or shift, scale (0): eight elements that every lane reads.
template <int DT>
struct Absent;
template <> struct Absent<MXF8_BF16> { static constexpr uint32_t one = 0x3f803f80u; };
template <> struct Absent<MXF8_F16> { static constexpr uint32_t one = 0x3c003c00u; };
template <> struct Absent<MXF8_F32> { static constexpr uint32_t one = 0x3f800000u; };
__device__ const uint32_t absent_zero[8] = {};
template <int DT>
__device__ const uint32_t absent_one[8] = {Absent<DT>::one, Absent<DT>::one, Absent<DT>::one, Absent<DT>::one,
                                           Absent<DT>::one, Absent<DT>::one, Absent<DT>::one, Absent<DT>::one};

// Waves per SIMD that the registers are cut for: as many as hold a row and its operands without a spill (20280 x
// 3072 in bf16, six chunks: four waves with spills 104.2 us, three without 91.5; with both norm weights 1.7
// times as long with spills).
constexpr int min_waves(int dt, int chunks, bool weights) {
  return dt == MXF8_F32 ? (chunks > 3 || (weights && chunks > 2) ? 2 : 4) : chunks > 4 ? 3 : 4;
}

// NT threads per row (below 256: 256 / NT rows per block), NC chunks of 8 elements per thread, of which the last one alone may
// lie past the row's end.  TAIL_BACK (C % 8 != 0): the row's last chunk starts 8 elements before its end instead; what
// it shares with the chunk before it counts there, and is stored twice alike (10166 x 2730: 46.5 us, with the elements
// behind the last whole chunk one by one 50.3; 2728 channels 45.8).  TAIL_SHORT (C < 8): one chunk of C
// elements.  WEIGHTS: branch_weight or weight may be there.
//
// What bounds it is memory, as long as the loads do not wait for each other: an operand's chunks are loaded with
// no condition between them (an absent operand is eight constants that every lane reads), the row's and the
// gate's first, the modulation's before the sums.  20280 x 3072 in bf16: 86-88 us, 498 MB at 5.7 TB/s, with e4m3 codes
// 79 (5.5 TB/s), with mxfp4 codes 76 (5.4); with norms before and behind 90, 83 and 81.
enum { TAIL_NONE, TAIL_BACK, TAIL_SHORT };

template <int DT, int NT, int NC, int QM, int TAIL, bool WEIGHTS>
__global__ __launch_bounds__(NT > 256 ? NT : 256, min_waves(DT, NC, WEIGHTS)) void block_norm_kernel(const BlockNormArgs a) {
  __shared__ float red[NT > 64 ? NT / 64 : 1];
  const int t = threadIdx.x % NT;
  const int sub = NT < 64 ? threadIdx.x / NT : __builtin_amdgcn_readfirstlane(threadIdx.x / NT);  // row of the block
  const int m = blockIdx.x * ((NT > 256 ? NT : 256) / NT) + sub;
  if (m >= a.M) return;  // (all lanes of a row; whole blocks where a block is a row)
  const int b = m / a.S, s = m - b * a.S, span = s / a.span;
  const int C = a.C;
  const int at_last = 8 * ((NC - 1) * NT + t);
  const bool whole = at_last < C;  // the last chunk is there
  // chunk c: elements [at, at + 8) of the row, of which [lo, hi) of the last one are not another chunk's
  const int back = TAIL == TAIL_BACK ? min(at_last, C - 8) : at_last;
  const int lo = at_last - back, hi = TAIL == TAIL_SHORT ? C : 8;
  auto at = [&](int c) { return c < NC - 1 ? 8 * (c * NT + t) : back; };
  auto own = [&](int c, int i) { return TAIL == TAIL_NONE || c < NC - 1 || (i >= lo && i < hi); };
  typedef typename Elem<DT>::T T;
  const bool has_br = a.branch != nullptr, has_g = a.gate != nullptr, has_sh = a.shift != nullptr,
             has_sc = a.scale != nullptr;
  const T* const zero = reinterpret_cast<const T*>(absent_zero);
  const T* const one = reinterpret_cast<const T*>(absent_one<DT>);
  const T* const x = static_cast<const T*>(a.x) + (int64_t)b * a.x_b + (int64_t)s * a.x_s;
  const T* const br = has_br ? static_cast<const T*>(a.branch) + (int64_t)b * a.br_b + (int64_t)s * a.br_s : zero;
  const T* const g = has_g ? static_cast<const T*>(a.gate) + (int64_t)b * a.g_b + (int64_t)span * a.g_s : one;
  const T* const sh = has_sh ? static_cast<const T*>(a.shift) + (int64_t)b * a.sh_b + (int64_t)span * a.sh_s : zero;
  const T* const sc = has_sc ? static_cast<const T*>(a.scale) + (int64_t)b * a.sc_b + (int64_t)span * a.sc_s : zero;
  const bool has_bw = a.branch_weight != nullptr, has_w = a.weight != nullptr;
  const T* const bw = has_bw ? static_cast<const T*>(a.branch_weight) : one;
  const T* const w = has_w ? static_cast<const T*>(a.weight) : one;
  const int64_t ro = (int64_t)m * C;

  auto load = [&](auto& v, const T* p, bool there) {
    const uint32_t first = there ? 8 * t * sizeof(T) : 0, step = there ? 8 * NT * sizeof(T) : 0;
#pragma unroll
    for (int c = 0; c < NC - 1; ++c) v[c].load_off(p, first + c * step);
    v[NC - 1].zero();
    if (TAIL == TAIL_SHORT && there) {
      if (whole) v[NC - 1].load_part(p, 0, hi);
    } else if (whole) {
      v[NC - 1].load_off(p, TAIL == TAIL_BACK ? (there ? back * sizeof(T) : 0) : first + (NC - 1) * step);
    }
  };
  // The scheduler fills waits with whatever follows, and unpacking the operands of a later phase early costs it
  // the registers of four waves.
  auto phase = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  Raw8<DT> xv[NC], bv[NC], gv[NC];
  load(xv, x, true);
  load(bv, br, has_br);
  load(gv, g, has_g);
  Raw8<DT> wv[WEIGHTS ? NC : 1];
  float post = 1.0f;
  constexpr int PARTS = NT == 64 && NC > 2 ? (NC < 4 ? NC : 4) : 1;
  if constexpr (WEIGHTS) {
    load(wv, bw, has_bw);
    if (has_bw) {
      float ss[PARTS] = {};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float f[8];
        bv[c].get(f);
        bv[c].hide();
#pragma unroll
        for (int i = 0; i < 8; ++i) ss[c % PARTS] = own(c, i) ? __builtin_fmaf(f[i], f[i], ss[c % PARTS]) : ss[c % PARTS];
        __builtin_amdgcn_sched_barrier(0);
      }
      post = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(row_sum<NT, PARTS>(ss, red), (float)C) + a.eps));
    }
  }
  float r[NC][8];
  float sum[PARTS] = {};
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float f[8], h[8], u[8];
    bv[c].get(u);
    xv[c].get(f);
    gv[c].get(h);
    if constexpr (WEIGHTS) {
      float k[8];
      wv[c].get(k);
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] *= post * k[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      r[c][i] = __builtin_fmaf(h[i], u[i], f[i] * a.residual_scale);
      sum[c % PARTS] += own(c, i) ? r[c][i] : 0.0f;
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // the next norm's modulation, in flight over the sums
  phase();
  Raw8<DT> sv[NC], hv[NC];
  load(sv, sc, has_sc);
  load(hv, sh, has_sh);
  auto put = [&](const Raw8<DT>& o, void* to, int c) {
    if (c == NC - 1 && !whole) return;
    if (TAIL == TAIL_SHORT)
      o.store_part(to, ro, hi);
    else
      o.stream(to, ro + at(c));
  };
  if (has_br) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      Raw8<DT> o;
      o.set(r[c]);
      put(o, a.r, c);
    }
  }
  phase();
  const float mean = a.layer ? __fdiv_rn(row_sum<NT, PARTS>(sum, red), (float)C) : 0.0f;
  float ss[PARTS] = {};
#pragma unroll
  for (int c = 0; c < NC; ++c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r[c][i] -= mean;
    if (c == NC - 1 && !whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[c][i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss[c % PARTS] = own(c, i) ? __builtin_fmaf(r[c][i], r[c][i], ss[c % PARTS]) : ss[c % PARTS];
  }
  const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(row_sum<NT, PARTS>(ss, red), (float)C) + a.eps));
  phase();
  if constexpr (WEIGHTS) load(wv, w, has_w);
  float amax = 0.0f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float f[8], h[8];
    sv[c].get(f);
    hv[c].get(h);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[c][i] *= rstd;
    if constexpr (WEIGHTS) {
      float k[8];
      wv[c].get(k);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[c][i] *= k[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) r[c][i] = __builtin_fmaf(r[c][i], 1.0f + f[i], h[i]);
    Raw8<DT> o;
    o.set(r[c]);
    if (QM == MXF8_QUANT_NONE || a.y) put(o, a.y, c);
    if constexpr (QM != MXF8_QUANT_NONE) o.get(r[c]);  // y as it is stored (0 past the row's end)
    if constexpr (QM == MXF8_QUANT_E4M3) {
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, TAIL == TAIL_SHORT && i >= hi ? 0.0f : fabsf(r[c][i]));
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  if constexpr (QM == MXF8_QUANT_E4M3) {
    const float s8 = e4m3_scale(row_max<NT>(amax, red));
    const float inv = __fdiv_rn(1.0f, s8);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = clamp448(div_by_scale(r[c][i], s8, inv));
      struct __attribute__((packed, aligned(1))) W2 {
        uint32_t w[2];
      } const q = {{cvt4_e4m3(f[0], f[1], f[2], f[3]), cvt4_e4m3(f[4], f[5], f[6], f[7])}};
      if (c == NC - 1 && !whole) continue;
      if constexpr (TAIL == TAIL_SHORT) {
#pragma unroll
        for (int i = 0; i < 7; ++i)
          if (i < hi) a.codes[ro + i] = (uint8_t)(q.w[i >> 2] >> (8 * (i & 3)));
      } else {
        *reinterpret_cast<W2*>(a.codes + ro + at(c)) = q;
      }
    }
    if (t == 0) a.row_scale[m] = s8;
  }
  if constexpr (QM == MXF8_QUANT_MXFP4) {
    const int padded = (int)mx_slabs(C) * MX_BLOCK * MX_SLAB;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const uint32_t byte = mx_scale_byte(mx_block_absmax(r[c]));
      if (c < NC - 1 || whole) *reinterpret_cast<uint32_t*>(a.codes + (int64_t)m * (C / 2) + at(c) / 2) = mx_codes8(r[c], byte);
      if (at(c) < padded && (t & 3) == 0)
        a.mx_scales[mx_scale_at(at(c) / MX_BLOCK, m, a.M)] = (uint8_t)(at(c) < C ? byte : 127u);
    }
  }
}

template <int DT, int NT, int NC, int QM>
static int launch_block_norm_nc(const BlockNormArgs& a, hipStream_t st) {
  const char* what = "gated_residual_norm";
  constexpr int block = NT > 256 ? NT : 256;
  const int64_t blocks = cdiv(a.M, block / NT);
  if (!grid_fits(blocks, block)) return set_error(MXF8_EINVAL, "%s: shape too large", what);
  const dim3 grid((unsigned)blocks);
  const bool weights = a.branch_weight || a.weight;
  if constexpr (QM != MXF8_QUANT_MXFP4) {
    if (a.C % 8) {
      if constexpr (NT == 8) {
        if (a.C < 8) {
          block_norm_kernel<DT, NT, NC, QM, TAIL_SHORT, true><<<grid, block, 0, st>>>(a);
          return check_launch(what);
        }
      }
      block_norm_kernel<DT, NT, NC, QM, TAIL_BACK, true><<<grid, block, 0, st>>>(a);
      return check_launch(what);
    }
  }
  if (weights)
    block_norm_kernel<DT, NT, NC, QM, TAIL_NONE, true><<<grid, block, 0, st>>>(a);
  else
    block_norm_kernel<DT, NT, NC, QM, TAIL_NONE, false><<<grid, block, 0, st>>>(a);
  return check_launch(what);
}

template <int DT, int QM>
static int launch_block_norm(const BlockNormArgs& a, hipStream_t st) {
  // chunks of a row (with mxfp4, of the padded row whose scale bytes are written)
  int64_t chunks = cdiv(a.C, 8);
  if (QM == MXF8_QUANT_MXFP4) chunks = mx_slabs(a.C) * MX_BLOCK * MX_SLAB / 8;
  // One wave per row where a lane has two chunks at most, or up to six (three in fp32) once there are rows for every
  // wave that fits; else four waves per row, whose parts of a row wait for each other at the sums but load it
  // at once.  3072 channels in bf16, one wave / four: 1 token 4.2 / 3.9 us, 512 6.1 / 5.2, 8192 40.4 / 40.1,
  // 20280 88.8 / 92.0; 1024 channels: 512 tokens 4.1 / 4.4, 10166 16.0 / 23.4.
  const bool wave = chunks <= 128 || (chunks <= (DT == MXF8_F32 ? 192 : 384) && a.M >= 8192);
#define MXF8_BN(NT, NC) \
  case NC: return launch_block_norm_nc<DT, NT, NC, QM>(a, st);
  // Short rows share a wave: 51597 x 33 30.0 -> 8.2 us, 20000 x 256 13.2 -> 10.0.
  if (chunks <= 32) {
    return chunks <= 8    ? launch_block_norm_nc<DT, 8, 1, QM>(a, st)
           : chunks <= 16 ? launch_block_norm_nc<DT, 16, 1, QM>(a, st)
                          : launch_block_norm_nc<DT, 32, 1, QM>(a, st);
  } else if (wave) {
    switch (cdiv(chunks, 64)) {
      MXF8_BN(64, 1) MXF8_BN(64, 2) MXF8_BN(64, 3)
      default:
        if constexpr (DT != MXF8_F32) {
          switch (cdiv(chunks, 64)) { MXF8_BN(64, 4) MXF8_BN(64, 5) MXF8_BN(64, 6) }
        }
    }
  } else if (chunks <= 4 * 256) {
    switch (cdiv(chunks, 256)) { MXF8_BN(256, 1) MXF8_BN(256, 2) MXF8_BN(256, 3) MXF8_BN(256, 4) }
  } else {
    switch (cdiv(chunks, 512)) { MXF8_BN(512, 3) MXF8_BN(512, 4) }
  }
#undef MXF8_BN
  return set_error(MXF8_EINVAL, "gated_residual_norm: no kernel for C=%d", a.C);
}

}  // namespace mxf8

using namespace mxf8;

extern "C" int mxf8_gated_residual_norm(const void* x, int64_t x_batch, int64_t x_token, const void* branch,
                                        int64_t br_batch, int64_t br_token, int dtype, int64_t B, int64_t S, int64_t C,
                                        const void* gate, int64_t g_batch, int64_t g_span, const void* shift,
                                        int64_t sh_batch, int64_t sh_span, const void* scale, int64_t sc_batch,
                                        int64_t sc_span, int64_t spans, const void* branch_weight, const void* weight,
                                        int layer, float eps, float residual_scale, int quant, void* r, void* y,
                                        uint8_t* codes, void* scales, hipStream_t stream) {
  const char* what = "gated_residual_norm";
  if (B < 0 || S < 0 || C <= 0) return set_error(MXF8_EINVAL, "%s: bad shape", what);
  if (C > 16384) return set_error(MXF8_EINVAL, "%s: C=%lld exceeds 16384", what, (long long)C);
  if (dtype != MXF8_BF16 && dtype != MXF8_F16 && dtype != MXF8_F32)
    return set_error(MXF8_EINVAL, "%s: bad dtype %d", what, dtype);
  if (quant < MXF8_QUANT_NONE || quant > MXF8_QUANT_MXFP4) return set_error(MXF8_EINVAL, "%s: bad quantization %d", what, quant);
  if (quant == MXF8_QUANT_MXFP4 && C % MX_BLOCK)
    return set_error(MXF8_EINVAL, "%s: C=%lld must be a multiple of 32 for 4-bit blocks", what, (long long)C);
  if (!(eps >= 0.0f)) return set_error(MXF8_EINVAL, "%s: eps must be >= 0", what);
  if (spans < 1 || S % spans) return set_error(MXF8_EINVAL, "%s: %lld spans do not divide S=%lld", what,
                                               (long long)spans, (long long)S);
  if (B > (1 << 24) || S > (1 << 30) || B * S > 0x7fffffff) return set_error(MXF8_EINVAL, "%s: shape too large", what);
  if (B * S == 0) return MXF8_OK;
  if (!x || (branch && !r) || (quant == MXF8_QUANT_NONE && !y) || (quant != MXF8_QUANT_NONE && (!codes || !scales)))
    return set_error(MXF8_EINVAL, "%s: null pointer", what);
  if (!branch && (gate || branch_weight))
    return set_error(MXF8_EINVAL, "%s: gate and branch_weight need a branch", what);
  if (quant == MXF8_QUANT_MXFP4 && (uintptr_t)codes % 4) return set_error(MXF8_EINVAL, "%s: codes must be 4-byte aligned", what);
  BlockNormArgs a{};
  a.x = x, a.branch = branch, a.gate = gate, a.shift = shift, a.scale = scale;
  a.branch_weight = branch_weight, a.weight = weight;
  a.r = branch ? r : nullptr, a.y = y, a.codes = codes;
  a.row_scale = static_cast<float*>(scales);
  a.mx_scales = static_cast<uint8_t*>(scales);
  a.x_b = x_batch, a.x_s = x_token, a.br_b = br_batch, a.br_s = br_token;
  a.g_b = g_batch, a.g_s = g_span, a.sh_b = sh_batch, a.sh_s = sh_span, a.sc_b = sc_batch, a.sc_s = sc_span;
  a.S = (int)S, a.M = (int)(B * S), a.span = (int)(S / spans), a.C = (int)C, a.layer = layer != 0;
  a.eps = eps, a.residual_scale = residual_scale;
#define MXF8_CASE(DT)                                                        \
  case DT:                                                                   \
    return quant == MXF8_QUANT_NONE  ? launch_block_norm<DT, MXF8_QUANT_NONE>(a, stream)   \
           : quant == MXF8_QUANT_E4M3 ? launch_block_norm<DT, MXF8_QUANT_E4M3>(a, stream)    \
                              : launch_block_norm<DT, MXF8_QUANT_MXFP4>(a, stream);
  switch (dtype) {
    MXF8_CASE(MXF8_BF16)
    MXF8_CASE(MXF8_F16)
    default: break;
    MXF8_CASE(MXF8_F32)
  }
#undef MXF8_CASE
  return set_error(MXF8_EINVAL, "%s: bad dtype %d", what, dtype);
}
