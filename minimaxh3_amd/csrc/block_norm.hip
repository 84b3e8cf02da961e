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
  int64_t S, M;
  int span;  // tokens per modulation row
  int C, layer;
  float eps, residual_scale;
};

// Sum over the NT threads that hold a row, in every one of them.
template <int NT>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = wave_sum(v);
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
  v = wave_max(v);
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

// NT threads per row (64: four rows per block), NC chunks of 8 elements per thread; with TAIL, the C % 8 elements
// behind the row's last whole chunk are one element each of its first threads.
template <int DT, int NT, int NC, int QM, bool TAIL>
__global__ __launch_bounds__(256) void block_norm_kernel(const BlockNormArgs a) {
  __shared__ float red[4];
  const int t = threadIdx.x % NT;
  const int64_t m = (int64_t)blockIdx.x * (256 / NT) + threadIdx.x / NT;
  if (m >= a.M) return;  // (whole waves; whole blocks where a block is a row)
  const int64_t b = m / a.S, s = m - b * a.S, span = s / a.span;
  const int C = a.C, C8 = C & ~7;
  auto at = [&](int c) { return 8 * (c * NT + t); };  // chunk c: elements [at, at + 8) of the row, if below C8
  const int te = C8 + t;                               // the tail element
  const bool tail = TAIL && te < C;
  const int64_t xo = b * a.x_b + s * a.x_s, bo = b * a.br_b + s * a.br_s, ro = m * C;
  const int64_t go = b * a.g_b + span * a.g_s, sho = b * a.sh_b + span * a.sh_s, sco = b * a.sc_b + span * a.sc_s;

  Raw8<DT> xv[NC], bv[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    xv[c].zero();
    bv[c].zero();
    if (at(c) < C8) {
      xv[c].load(a.x, xo + at(c));
      if (a.branch) bv[c].load(a.branch, bo + at(c));
    }
  }
  float rt = 0.0f, bt = 0.0f;
  if (tail) {
    rt = load1<DT>(a.x, xo + te) * a.residual_scale;
    if (a.branch) bt = load1<DT>(a.branch, bo + te);
  }
  float post = 1.0f;
  if (a.branch_weight) {
    float ss = bt * bt;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float f[8];
      bv[c].get(f);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(f[i], f[i], ss);
    }
    post = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(row_sum<NT>(ss, red), (float)C) + a.eps));
  }
  float r[NC][8];
  float sum = 0.0f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    xv[c].get(r[c]);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[c][i] *= a.residual_scale;
    if (at(c) < C8 && a.branch) {
      float u[8], f[8];
      Raw8<DT> w;
      bv[c].get(u);
      if (a.branch_weight) {
        w.load(a.branch_weight, at(c));
        w.get(f);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] *= post * f[i];
      }
      if (a.gate) {
        w.load(a.gate, go + at(c));
        w.get(f);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[c][i] = __builtin_fmaf(f[i], u[i], r[c][i]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r[c][i] += u[i];
      }
      w.set(r[c]);
      w.store(a.r, ro + at(c));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += r[c][i];
  }
  if (tail && a.branch) {
    if (a.branch_weight) bt *= post * load1<DT>(a.branch_weight, te);
    rt = a.gate ? __builtin_fmaf(load1<DT>(a.gate, go + te), bt, rt) : rt + bt;
    store1<DT>(a.r, ro + te, rt);
  }
  if constexpr (TAIL) sum += rt;
  const float mean = a.layer ? __fdiv_rn(row_sum<NT>(sum, red), (float)C) : 0.0f;
  float ss = 0.0f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (at(c) < C8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = r[c][i] - mean;
        ss = __builtin_fmaf(d, d, ss);
      }
    }
  }
  if (tail) ss = __builtin_fmaf(rt - mean, rt - mean, ss);
  const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(row_sum<NT>(ss, red), (float)C) + a.eps));
  float amax = 0.0f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (at(c) < C8) {
      float f[8];
      Raw8<DT> w;
#pragma unroll
      for (int i = 0; i < 8; ++i) r[c][i] = (r[c][i] - mean) * rstd;
      if (a.weight) {
        w.load(a.weight, at(c));
        w.get(f);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[c][i] *= f[i];
      }
      if (a.scale) {
        w.load(a.scale, sco + at(c));
        w.get(f);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[c][i] *= 1.0f + f[i];
      }
      if (a.shift) {
        w.load(a.shift, sho + at(c));
        w.get(f);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[c][i] += f[i];
      }
      w.set(r[c]);
      if (QM == MXF8_QUANT_NONE || a.y) w.store(a.y, ro + at(c));
      if constexpr (QM != MXF8_QUANT_NONE) w.get(r[c]);  // y as it is stored
      if constexpr (QM == MXF8_QUANT_E4M3) {
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(r[c][i]));
      }
    }
  }
  if (tail) {
    rt = (rt - mean) * rstd;
    if (a.weight) rt *= load1<DT>(a.weight, te);
    if (a.scale) rt *= 1.0f + load1<DT>(a.scale, sco + te);
    if (a.shift) rt += load1<DT>(a.shift, sho + te);
    if (QM == MXF8_QUANT_NONE || a.y) store1<DT>(a.y, ro + te, rt);
    rt = round1<DT>(rt);
    amax = fmaxf(amax, fabsf(rt));
  }
  if constexpr (QM == MXF8_QUANT_E4M3) {
    const float sc = e4m3_scale(row_max<NT>(amax, red));
    const float inv = __fdiv_rn(1.0f, sc);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (at(c) < C8) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = clamp448(div_by_scale(r[c][i], sc, inv));
        struct __attribute__((packed, aligned(1))) W2 {
          uint32_t w[2];
        };
        *reinterpret_cast<W2*>(a.codes + ro + at(c)) =
            W2{{cvt4_e4m3(f[0], f[1], f[2], f[3]), cvt4_e4m3(f[4], f[5], f[6], f[7])}};
      }
    }
    if (tail) a.codes[ro + te] = (uint8_t)(cvt2_e4m3(clamp448(div_by_scale(rt, sc, inv)), 0.0f) & 0xff);
    if (t == 0) a.row_scale[m] = sc;
  }
  if constexpr (QM == MXF8_QUANT_MXFP4) {
    const int padded = (int)mx_slabs(C) * MX_BLOCK * MX_SLAB;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const uint32_t byte = mx_scale_byte(mx_block_absmax(r[c]));
      if (at(c) < C) *reinterpret_cast<uint32_t*>(a.codes + m * (C / 2) + at(c) / 2) = mx_codes8(r[c], byte);
      if (at(c) < padded && (t & 3) == 0)
        a.mx_scales[mx_scale_at(at(c) / MX_BLOCK, m, a.M)] = (uint8_t)(at(c) < C ? byte : 127u);
    }
  }
}

template <int DT, int QM>
static int launch_block_norm(const BlockNormArgs& a, hipStream_t st) {
  // chunks of a row (with mxfp4, of the padded row whose scale bytes are written)
  const int64_t chunks = QM == MXF8_QUANT_MXFP4 ? mx_slabs(a.C) * MX_BLOCK * MX_SLAB / 8 : cdiv(a.C, 8);
  // One wave per row up to 8 chunks a lane, once there are enough rows to fill the chip with them.
  const bool wave = chunks <= 512 && a.M >= 4096;
  const int64_t per = cdiv(chunks, wave ? 64 : 256);
  const dim3 grid((unsigned)cdiv(a.M, wave ? 4 : 1));
  const bool tail = a.C % 8 != 0;
#define MXF8_BN(NT, NC)                                                                              \
  do {                                                                                               \
    if constexpr (QM != MXF8_QUANT_MXFP4) {                                                                  \
      if (tail) {                                                                                    \
        block_norm_kernel<DT, NT, NC, QM, true><<<grid, 256, 0, st>>>(a);                            \
        break;                                                                                       \
      }                                                                                              \
    }                                                                                                \
    block_norm_kernel<DT, NT, NC, QM, false><<<grid, 256, 0, st>>>(a);                               \
  } while (0)
  if (wave) {
    if (per <= 1) MXF8_BN(64, 1);
    else if (per <= 2) MXF8_BN(64, 2);
    else if (per <= 4) MXF8_BN(64, 4);
    else if (per <= 6) MXF8_BN(64, 6);
    else MXF8_BN(64, 8);
  } else {
    if (per <= 1) MXF8_BN(256, 1);
    else if (per <= 2) MXF8_BN(256, 2);
    else if (per <= 4) MXF8_BN(256, 4);
    else MXF8_BN(256, 8);
  }
#undef MXF8_BN
  return check_launch("gated_residual_norm");
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
  a.S = S, a.M = B * S, a.span = (int)(S / spans), a.C = (int)C, a.layer = layer != 0;
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
