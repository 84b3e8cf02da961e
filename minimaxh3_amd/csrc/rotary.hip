// Rotary positions over several axes (time, height, width, ...): the table of cos / sin pairs, and the rotation
// of the query and key parts of a projection with the per-head RMS norm before it.
//
//   table[s, j] = (cos a, sin a), a = pos[s, axis(j)] * theta^(-2 i / d_axis): pair j is the i-th of its axis,
//                 whose d_axis channels hold d_axis / 2 pairs
//   y = x / sqrt(mean(x^2) + eps) * w  (per head; without weights y = x)
//   (u, v) = (a cos - b sin, a sin + b cos) for the pairs (a, b) of y: channels (2 j, 2 j + 1), or (j, j + P)
//            with P pairs; channels from 2 P on stay as they are
// Everything is fp32 between the load and the one rounding at the store.
#include <type_traits>

#include "common.h"
#include "rowio.h"

namespace mxf8 {

constexpr int ROT_MAX_AXES = 4, ROT_MAX_PAIRS = 256;

struct RotAxes {
  int first[ROT_MAX_AXES + 1];  // first pair of each axis, and the number of pairs
  double log2_theta;
};

// Position i from the uniform `base` on, of pos_type PT.
template <int PT>
__device__ __forceinline__ double rot_pos(const void* p, int64_t base, int i) {
  if constexpr (PT == 0)
    return (static_cast<const float*>(p) + base)[i];
  else if constexpr (PT == 1)
    return (static_cast<const double*>(p) + base)[i];
  else if constexpr (PT == 2)
    return (static_cast<const int*>(p) + base)[i];
  else
    return (double)(static_cast<const int64_t*>(p) + base)[i];
}

// cos and sin of `rev` revolutions.  The angle is reduced in fp64 to an eighth of a turn either way, exactly, so
// positions in the millions lose nothing; there the Taylor series to the 9th and 10th power are within 2^-26.
__device__ __forceinline__ v2f rot_cos_sin(double rev) {
  const double turn = rev - __builtin_rint(rev);  // -1/2 .. 1/2
  const float q = __builtin_rintf(4.0f * (float)turn);  // -2 .. 2 (either neighbour of a tie will do)
  const float x = (float)(__builtin_fma((double)q, -0.25, turn) * 6.283185307179586);
  const float x2 = x * x;
  float s = __builtin_fmaf(x2, 2.7557319e-6f, -1.9841270e-4f);
  s = __builtin_fmaf(x2, s, 8.3333333e-3f);
  s = __builtin_fmaf(x2, s, -1.6666667e-1f);
  s = __builtin_fmaf(x * x2, s, x);
  float c = __builtin_fmaf(x2, -2.7557319e-7f, 2.4801587e-5f);
  c = __builtin_fmaf(x2, c, -1.3888889e-3f);
  c = __builtin_fmaf(x2, c, 4.1666667e-2f);
  c = __builtin_fmaf(x2, c, -0.5f);
  c = __builtin_fmaf(x2, c, 1.0f);
  const int k = (int)q & 3;
  const float cc = k & 1 ? s : c, ss = k & 1 ? c : s;
  return v2f{k == 1 || k == 2 ? -cc : cc, k >= 2 ? -ss : ss};
}

// A block makes the pairs of `rows` consecutive tokens; the frequencies (in turns per position) are made once
// per block, in LDS.  Some 59 vector instructions a pair, four of them fp64, bound it: 20280 x 64 pairs 6.3 us (1.7 TB/s;
// a call takes the host 6), 77648 x 64 13.4 us (3.0 TB/s).
template <int PT>
__global__ __launch_bounds__(256) void rotary_table_kernel(const void* __restrict__ pos, int64_t n, int axes,
                                                           const RotAxes ax, int rows, float* __restrict__ table) {
  __shared__ double freq[ROT_MAX_PAIRS];
  __shared__ uint8_t axis[ROT_MAX_PAIRS];
  const int P = ax.first[axes];
  for (int j = threadIdx.x; j < P; j += 256) {
    int a = 0;
#pragma unroll
    for (int i = 1; i < ROT_MAX_AXES; ++i) a += i < axes && j >= ax.first[i];
    int lo = 0, hi = 0;
#pragma unroll
    for (int i = 0; i < ROT_MAX_AXES; ++i)
      if (i == a) lo = ax.first[i], hi = ax.first[i + 1];
    freq[j] = exp2(-ax.log2_theta * (double)(j - lo) / (double)(hi - lo)) * 0.15915494309189535;
    axis[j] = (uint8_t)a;
  }
  __syncthreads();
  const int64_t t0 = (int64_t)blockIdx.x * rows;
  const int cnt = (int)min((int64_t)rows, n - t0) * P;
  // entry e = t P + j, 256 further each time: t and j move by the same amounts but for a carry
  const int dt = 256 / P, dj = 256 - dt * P;
  int t = threadIdx.x / P, j = threadIdx.x - t * P;
  int row = t * axes;  // of the block's first token's positions
  float* o = table + (t0 * P + threadIdx.x) * 2;
  for (int e = threadIdx.x; e < cnt; e += 256, o += 512) {
    *reinterpret_cast<v2f*>(o) = rot_cos_sin(rot_pos<PT>(pos, t0 * axes, row + axis[j]) * freq[j]);
    row += dt * axes;
    j += dj;
    if (j >= P) j -= P, row += axes;
  }
}

struct RotArgs {
  const void *x[2], *w[2];  // q and k, and their norms' weights (null: no norm)
  void* o[2];
  int64_t xs[2][3], os[2][3];  // strides of batch, head, token (channels are contiguous)
  int heads[2];
  const float* table;
  int64_t table_batch;  // table elements per batch item (0: shared)
  int64_t S;
  int D, P, B;
  int steps[2], per;  // head steps of q and k, and how many one wave takes
  float eps, inv_d;
};

// a x + b y.  Which product the compiler fuses with the sum is its choice at every place, and with it the last bit:
// written out, a token's result does not depend on where in the unrolled steps its head falls.
__device__ __forceinline__ float turn(float a, float x, float b, float y) { return __builtin_fmaf(a, x, b * y); }

// One wave per token and span of head steps: L lanes hold a head (8 channels each), so a step moves 64 / L heads,
// 16 bytes a lane.  The token's cos / sin and the norm's weights stay in registers over the heads, and the
// next ROT_UNROLL steps' loads are in flight together.
//
// HEAD_FULL: a head fills its lanes (D = 8 L); HEAD_CHUNKS: whole chunks of 8 channels, and half-split pairs at the
// same place of two lanes' chunks (P % 8 == 0); HEAD_ANY: the last chunk may be cut, and half-split partners
// come through LDS.
//
// Bound by memory: 20280 tokens x (24 + 24) heads x 128 in bf16, 509 MB, 92 us (5.5 TB/s), the same without the
// norm; one step at a time 96.5, with stores that stay in the caches 100.
constexpr int ROT_UNROLL = 6;
enum { HEAD_FULL, HEAD_CHUNKS, HEAD_ANY };

template <int DT, int L, bool INTERLEAVED, int MODE>
__global__ __launch_bounds__(256) void rotate_qk_kernel(const RotArgs a) {
  constexpr int G = 64 / L, ES = DT == MXF8_F32 ? 4 : 2;
  __shared__ float exchange[MODE == HEAD_ANY && !INTERLEAVED ? 4 * 512 : 1];
  const int lane = threadIdx.x & 63, l = lane % L, hg = lane / L;
  const int64_t token = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (token >= a.S * a.B) return;
  const int b = (uint32_t)token / (uint32_t)a.S;
  const int64_t s = token - (int64_t)b * a.S;
  const int c0 = 8 * l;                       // this lane's channels
  const bool there = MODE == HEAD_FULL || c0 < a.D;  // any of them
  const int n = MODE == HEAD_ANY ? min(max(a.D - c0, 0), 8) : 8;  // how many, if any
  const float2* tab = reinterpret_cast<const float2*>(a.table + b * a.table_batch) + s * a.P;
  constexpr int NP = INTERLEAVED ? 4 : 8;
  float co[NP], si[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int c = INTERLEAVED ? c0 / 2 + i : c0 + i;
    const int j = INTERLEAVED || c < a.P ? c : c - a.P;  // (half-split: the second halves' pairs again)
    const bool turns = j < a.P;
    float2 t = make_float2(1.0f, 0.0f);
    if (turns) t = tab[j];
    co[i] = t.x;
    si[i] = INTERLEAVED || c >= a.P ? t.y : -t.y;
  }
  // half-split partner: channel c +- P is in lane l +- P / 8, at the same place of its eight as P % 8 == 0
  const int plane = (lane - l) + min(max(c0 < a.P ? l + a.P / 8 : l - a.P / 8, 0), L - 1);
  const int first = blockIdx.y * a.per, last = min(first + a.per, a.steps[0] + a.steps[1]);

  auto part = [&](auto p_tag) {
    constexpr int p = decltype(p_tag)::value;
    const int s0 = max(first - (p ? a.steps[0] : 0), 0), s1 = min(last - (p ? a.steps[0] : 0), a.steps[p]);
    if (s0 >= s1) return;
    const bool norm = a.w[p] != nullptr;
    Raw8<DT> wv, wp;
    wv.zero();
    if (norm && there) {
      if (MODE != HEAD_ANY || n == 8)
        wv.load(a.w[p], c0);
      else
        wv.load_part(a.w[p], c0, n);
    }
    wp = wv;
    if constexpr (!INTERLEAVED && MODE != HEAD_ANY) wp.from_lane(plane);
    const char* x = static_cast<const char*>(a.x[p]) + ((int64_t)b * a.xs[p][0] + s * a.xs[p][2]) * ES;
    char* o = static_cast<char*>(a.o[p]) + ((int64_t)b * a.os[p][0] + s * a.os[p][2]) * ES;
    // byte offsets of this lane's head and channels within a step; heads past the last one read it again
    const uint32_t xo = (uint32_t)(hg * a.xs[p][1] + (there ? c0 : 0)) * ES, oo = (uint32_t)(hg * a.os[p][1] + c0) * ES;
    const int in_last = a.heads[p] - (a.steps[p] - 1) * G;  // heads of the last step
    const uint32_t xo_last = (uint32_t)(min(hg, in_last - 1) * a.xs[p][1] + (there ? c0 : 0)) * ES;
    const int64_t xstep = a.xs[p][1] * G * ES, ostep = a.os[p][1] * G * ES;
    for (int st = s0; st < s1; st += ROT_UNROLL) {
      Raw8<DT> v[ROT_UNROLL];
#pragma unroll
      for (int u = 0; u < ROT_UNROLL; ++u)
        if (st + u < s1) {
          const uint32_t off = st + u + 1 == a.steps[p] ? xo_last : xo;
          if (MODE != HEAD_ANY || n == 8)
            v[u].load_off(x + (st + u) * xstep, off);
          else
            v[u].load_part(x + (st + u) * xstep + off, 0, n);
        }
#pragma unroll
      for (int u = 0; u < ROT_UNROLL; ++u) {
        if (st + u >= s1) break;
        float f[8], q[8];
        if (!there) v[u].zero();
        v[u].get(f);
        if constexpr (!INTERLEAVED && MODE != HEAD_ANY) {
          v[u].from_lane(plane);
          v[u].get(q);
        }
        if (norm) {
          float ss = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(f[i], f[i], ss);
          const float r = rsqrtf(__builtin_fmaf(lanes_sum<L>(ss), a.inv_d, a.eps));
          float k[8];
          wv.get(k);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] *= r * k[i];
          if constexpr (!INTERLEAVED && MODE != HEAD_ANY) {
            wp.get(k);
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] *= r * k[i];
          }
        }
        if constexpr (!INTERLEAVED && MODE == HEAD_ANY) {
          // (this wave's part of the exchange alone: LDS operations of a wave complete in order)
          float* mine = exchange + (threadIdx.x & ~63) * 8;
          *reinterpret_cast<v4f*>(mine + lane * 8) = v4f{f[0], f[1], f[2], f[3]};
          *reinterpret_cast<v4f*>(mine + lane * 8 + 4) = v4f{f[4], f[5], f[6], f[7]};
          __builtin_amdgcn_wave_barrier();
          const float* head = mine + hg * L * 8;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int c = c0 + i, j = c < a.P ? c + a.P : c - a.P;
            q[i] = head[c < 2 * a.P ? j : c];
          }
          __builtin_amdgcn_wave_barrier();
        }
        float y[8];
        if constexpr (INTERLEAVED) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[2 * i] = turn(f[2 * i], co[i], f[2 * i + 1], -si[i]);
            y[2 * i + 1] = turn(f[2 * i], si[i], f[2 * i + 1], co[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = turn(f[i], co[i], q[i], si[i]);
        }
        if (2 * a.P < a.D) {  // what passes through does so as it is: 0 times an infinity would make it NaN
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = c0 + i < 2 * a.P ? y[i] : f[i];
        }
        Raw8<DT> w;
        w.set(y);
        if (there && (st + u + 1 < a.steps[p] || hg < in_last)) {
          if (MODE != HEAD_ANY || n == 8)
            w.stream_off(o + (st + u) * ostep, oo);
          else
            w.store_part(o + (st + u) * ostep + oo, 0, n);
        }
      }
    }
  };
  part(std::integral_constant<int, 0>{});
  part(std::integral_constant<int, 1>{});
}

// Heads wider than a wave's 512 channels: one wave per head, element by element.
template <int DT, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotate_qk_any_kernel(const RotArgs a) {
  typedef typename Elem<DT>::T T;
  const int lane = threadIdx.x & 63;
  const int64_t rows = a.S * a.B * (a.heads[0] + a.heads[1]);
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int nh = a.heads[0] + a.heads[1];
  const int64_t token = row / nh, b = token / a.S, s = token - b * a.S;
  int h = (int)(row - token * nh);
  const int part = h >= a.heads[0];
  h -= part ? a.heads[0] : 0;
  const T* x = static_cast<const T*>(a.x[part]) + b * a.xs[part][0] + h * a.xs[part][1] + s * a.xs[part][2];
  T* o = static_cast<T*>(a.o[part]) + b * a.os[part][0] + h * a.os[part][1] + s * a.os[part][2];
  const T* w = static_cast<const T*>(a.w[part]);
  float r = 1.0f;
  if (w) {
    float ss = 0.0f;
    for (int c = lane; c < a.D; c += 64) {
      const float f = Elem<DT>::to_f32(x[c]);
      ss = __builtin_fmaf(f, f, ss);
    }
    r = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(wave_sum(ss), (float)a.D) + a.eps));
  }
  auto get = [&](int c) { return w ? Elem<DT>::to_f32(x[c]) * (r * Elem<DT>::to_f32(w[c])) : Elem<DT>::to_f32(x[c]); };
  auto put = [&](int c, float f) { store1<DT>(o, c, f); };
  const float2* tab = reinterpret_cast<const float2*>(a.table + b * a.table_batch) + s * a.P;
  for (int j = lane; j < a.P; j += 64) {
    const int c0 = INTERLEAVED ? 2 * j : j, c1 = INTERLEAVED ? 2 * j + 1 : j + a.P;
    const float2 t = tab[j];
    const float u = get(c0), v = get(c1);
    put(c0, turn(u, t.x, v, -t.y));
    put(c1, turn(u, t.y, v, t.x));
  }
  for (int c = 2 * a.P + lane; c < a.D; c += 64) put(c, get(c));
}

template <int DT, bool INTERLEAVED>
static int launch_rotate(RotArgs& a, hipStream_t st) {
  const char* what = "rotate_qk";
  const int64_t tokens = a.S * a.B;
  const int64_t blocks = cdiv(a.D > 512 ? tokens * (a.heads[0] + a.heads[1]) : tokens, 4);
  if (!grid_fits(blocks, 256)) return set_error(MXF8_EINVAL, "%s: shape too large", what);
  if (a.D > 512) {
    rotate_qk_any_kernel<DT, INTERLEAVED><<<dim3((unsigned)blocks), 256, 0, st>>>(a);
    return check_launch(what);
  }
  // Lanes per head: the 8-channel chunks of a head, up to a power of two.  A lane's offset within a step of 64 / L
  // heads is 32 bits of bytes; heads that lie too far apart for that take a wave each, with the same result bit for bit
  // (the idle lanes add zeros to the norm's sum).  24 heads of 128 as [B, H, S, D] in memory, bf16, 140000 tokens: 337 us
  // (5.3 TB/s; as the views of a projection 315).  4 heads of 64, 4.6 million tokens in one step / 5.2 million, past
  // the 32 bits, a wave each: 2569 us (2.3 TB/s) / 3524 (1.9).
  int L = 8;
  while (L * 8 < a.D) L *= 2;
  constexpr int64_t ES = DT == MXF8_F32 ? 4 : 2;
  for (int p = 0; p < 2; ++p)
    for (const int64_t hs : {a.xs[p][1], a.os[p][1]})
      if (a.heads[p] > 1 && (hs < 0 || hs > ((1LL << 32) / ES - 512) / 7)) L = 64;
  a.steps[0] = (int)cdiv(a.heads[0], 64 / L);
  a.steps[1] = (int)cdiv(a.heads[1], 64 / L);
  const int total = a.steps[0] + a.steps[1];
  // All heads of a token in one wave once that gives every SIMD two waves; fewer tokens split the heads.
  a.per = total;
  while (a.per > 1 && tokens * cdiv(total, a.per) < 2048) a.per = (a.per + 1) / 2;
  const dim3 grid((unsigned)blocks, (unsigned)cdiv(total, a.per));
  const bool any = a.D % 8 || (!INTERLEAVED && a.P % 8);
#define MXF8_CASE(LL)                                                                \
  case LL:                                                                           \
    if (any)                                                                         \
      rotate_qk_kernel<DT, LL, INTERLEAVED, HEAD_ANY><<<grid, 256, 0, st>>>(a);      \
    else if (a.D == 8 * LL)                                                          \
      rotate_qk_kernel<DT, LL, INTERLEAVED, HEAD_FULL><<<grid, 256, 0, st>>>(a);     \
    else                                                                             \
      rotate_qk_kernel<DT, LL, INTERLEAVED, HEAD_CHUNKS><<<grid, 256, 0, st>>>(a);   \
    break;
  switch (L) {
    MXF8_CASE(8)
    MXF8_CASE(16)
    MXF8_CASE(32)
    MXF8_CASE(64)
  }
#undef MXF8_CASE
  return check_launch(what);
}

}  // namespace mxf8

using namespace mxf8;

extern "C" int mxf8_rotary_table(const void* pos, int pos_type, int64_t n, int64_t axes, const int64_t* axis_dims,
                                 double theta, float* table, hipStream_t stream) {
  if (n < 0) return set_error(MXF8_EINVAL, "rotary_table: negative number of positions");
  if (axes < 1 || axes > ROT_MAX_AXES || !axis_dims)
    return set_error(MXF8_EINVAL, "rotary_table: 1 to %d axes expected", ROT_MAX_AXES);
  if (!(theta > 0.0) || !(theta < 1.0e30)) return set_error(MXF8_EINVAL, "rotary_table: theta must be positive");
  RotAxes ax{};
  ax.log2_theta = __builtin_log2(theta);
  int64_t P = 0;
  for (int64_t i = 0; i < axes; ++i) {
    if (axis_dims[i] <= 0 || axis_dims[i] % 2 || axis_dims[i] > 2 * ROT_MAX_PAIRS)
      return set_error(MXF8_EINVAL, "rotary_table: axis %lld has %lld channels (even numbers from 2 on expected)",
                       (long long)i, (long long)axis_dims[i]);
    ax.first[i] = (int)P;
    P += axis_dims[i] / 2;
    if (P > ROT_MAX_PAIRS) return set_error(MXF8_EINVAL, "rotary_table: more than %d pairs", ROT_MAX_PAIRS);
  }
  ax.first[axes] = (int)P;
  if (n == 0) return MXF8_OK;
  if (!pos || !table) return set_error(MXF8_EINVAL, "rotary_table: null pointer");
  if ((uintptr_t)table % 8) return set_error(MXF8_EINVAL, "rotary_table: table must be 8-byte aligned");
  // eight pairs a thread, fewer where that leaves compute units without a block
  int rows = (int)cdiv(2048, P);
  const int cus = device_cus();
  while (rows > 1 && cdiv(n, rows) < 4 * cus) rows = (rows + 1) / 2;
  if (!grid_fits(cdiv(n, rows), 256)) return set_error(MXF8_EINVAL, "rotary_table: too many positions");
  const dim3 grid((unsigned)cdiv(n, rows));
  switch (pos_type) {
    case 0: rotary_table_kernel<0><<<grid, 256, 0, stream>>>(pos, n, (int)axes, ax, rows, table); break;
    case 1: rotary_table_kernel<1><<<grid, 256, 0, stream>>>(pos, n, (int)axes, ax, rows, table); break;
    case 2: rotary_table_kernel<2><<<grid, 256, 0, stream>>>(pos, n, (int)axes, ax, rows, table); break;
    case 3: rotary_table_kernel<3><<<grid, 256, 0, stream>>>(pos, n, (int)axes, ax, rows, table); break;
    default: return set_error(MXF8_EINVAL, "rotary_table: bad position type %d", pos_type);
  }
  return check_launch("rotary_table");
}

extern "C" int mxf8_rotate_qk(const void* q, const int64_t q_strides[4], int64_t Hq, const void* k,
                              const int64_t k_strides[4], int64_t Hk, int dtype, int64_t B, int64_t S, int64_t D,
                              const float* table, int64_t table_batch_stride, int64_t P, const void* q_weight,
                              const void* k_weight, float eps, int interleaved, void* q_out,
                              const int64_t qo_strides[4], void* k_out, const int64_t ko_strides[4],
                              hipStream_t stream) {
  const char* what = "rotate_qk";
  if (B < 0 || S < 0 || Hq < 0 || Hk < 0 || D <= 0 || D > 4096) return set_error(MXF8_EINVAL, "%s: bad shape", what);
  if (P < 0 || 2 * P > D) return set_error(MXF8_EINVAL, "%s: %lld pairs do not fit D=%lld", what, (long long)P,
                                           (long long)D);
  if (dtype != MXF8_BF16 && dtype != MXF8_F16 && dtype != MXF8_F32)
    return set_error(MXF8_EINVAL, "%s: bad dtype %d", what, dtype);
  if (!(eps >= 0.0f)) return set_error(MXF8_EINVAL, "%s: eps must be >= 0", what);
  if (B > (1 << 24) || S > (1 << 30) || Hq > (1 << 14) || Hk > (1 << 14) || B * S > (1LL << 31) ||
      B * S * (Hq + Hk) > (1LL << 32))
    return set_error(MXF8_EINVAL, "%s: shape too large", what);
  if (B * S == 0 || Hq + Hk == 0) return MXF8_OK;
  if ((Hq && (!q || !q_out || !q_strides || !qo_strides)) || (Hk && (!k || !k_out || !k_strides || !ko_strides)) ||
      (P && !table))
    return set_error(MXF8_EINVAL, "%s: null pointer", what);
  if ((uintptr_t)table % 8 || table_batch_stride % 2) return set_error(MXF8_EINVAL, "%s: table must be 8-byte aligned", what);
  RotArgs a{};
  const void* xs[2] = {q, k};
  const void* ws[2] = {q_weight, k_weight};
  void* os[2] = {q_out, k_out};
  const int64_t* st[2] = {q_strides, k_strides};
  const int64_t* so[2] = {qo_strides, ko_strides};
  const int64_t heads[2] = {Hq, Hk};
  for (int p = 0; p < 2; ++p) {
    a.heads[p] = (int)heads[p];
    if (!heads[p]) continue;
    if ((D > 1 && (st[p][3] != 1 || so[p][3] != 1)))
      return set_error(MXF8_EINVAL, "%s: channels must be contiguous", what);
    a.x[p] = xs[p], a.w[p] = ws[p], a.o[p] = os[p];
    for (int i = 0; i < 3; ++i) a.xs[p][i] = st[p][i], a.os[p][i] = so[p][i];
  }
  a.table = table;
  a.table_batch = table_batch_stride;
  a.S = S, a.B = (int)B, a.D = (int)D, a.P = (int)P;
  a.eps = eps;
  a.inv_d = 1.0f / (float)D;
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return interleaved ? launch_rotate<DT, true>(a, stream) : launch_rotate<DT, false>(a, stream);
  };
  return dtype == MXF8_BF16  ? launch(std::integral_constant<int, MXF8_BF16>{})
         : dtype == MXF8_F16 ? launch(std::integral_constant<int, MXF8_F16>{})
                             : launch(std::integral_constant<int, MXF8_F32>{});
}
