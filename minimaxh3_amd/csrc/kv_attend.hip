// Attention over a paged e4m3 cache of keys and values.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij, p_ij = 2^x_ij, x_ij = scale log2(e) q_i . k_j, over the keys j that row i sees
//
// Keys and values are codes times a power of two for each page.  Codes become fp16 exactly and go into the fp16 matrix
// instructions; a key's power of two multiplies the score, and a value's, 2^e_j, goes into the exponent:
//   p'_ij = 2^(x_ij + e_j - m_i),  o_i = sum_j p'_ij code_j / sum_j p'_ij 2^-e_j
// with m_i 7 below a running maximum of x_ij + e_j, or up to 15 below the maximum that is to come.  So the row's largest p' is
// from 2^7 to 2^15 (fp16 ends at 65504) however the pages' sizes differ, and p' half step in fp16, 2^-11 of it or 2^-25, is
// all that the value product rounds.  What this comes to in an output: 2^-11 of sum p |v| / sum p, and where p 2^e is far
// below the row's largest, 2^-32 max(p 2^e) |code_j| / sum p for each such key j.  (With the largest at 1 to 2^8 it was 2^-25: of 20280
// keys 2^-22 as likely as one whose value is 0, it lost up to 18%, and 2^-26 all.)  bf16 queries are exact in fp16
// under a power of two per row, down to 2^-17 of the row's largest (the half step below is 2^-25 of it).
// (e4m3 probabilities would run twice as fast and be off by 2^-4, bf16 ones by 2^-8.)
//
// The products are made transposed, S' = K Q' and O' = V' P': then a lane holds one row's scores and outputs, the maximum
// and the sum run within lanes, and the probabilities are in the layout that the second product reads.
#include <type_traits>

#include "kv_cache.h"
#include "rowio.h"

namespace mxf8 {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));

struct AttendArgs {
  KvPages c;
  const void* q;
  void* o;
  int64_t qs[3], os[3];  // strides of batch, head, token
  const int32_t *lengths, *q_lengths;
  int B, S, G, R, causal;  // G heads a key head, R = S G rows of it: row i G + g is query i of head g
  float scale;             // times log2 e
  int splits;              // parts of the keys
  float *part, *stat;      // with more than one: sums [B, Hk, splits, R, D], and (maximum, sum of p) [.., 2]
};

constexpr float KV_LARGEST = 3.40282347e38f;
constexpr float KV_NONE = -KV_LARGEST;  // a maximum of no scores: none is below it
// p' of a row's largest so far is 2^7 when m follows it, and may grow to 2^15 before m follows again.
constexpr float KV_UP = 7.0f, KV_SLACK = 8.0f;

// ---- rows and splits -------------------------------------------------------------------
struct KvSeq {
  int len, n;  // keys and queries that are there
  int diag;    // keys that the last query sees under a causal mask: tokens that the table has no entries for count here
};
__device__ __forceinline__ KvSeq kv_seq(const AttendArgs& a, int b) {
  KvSeq s;
  s.diag = max(a.lengths[b], 0);
  s.len = kv_length(a.c, s.diag);
  s.n = a.q_lengths ? min(max(a.q_lengths[b], 0), a.S) : a.S;
  return s;
}
// How many keys query i of s.n sees under a causal mask.
__device__ __forceinline__ int kv_seen(KvSeq s, int i) { return min(max(s.diag - (s.n - 1 - i), 0), s.len); }
// How many keys row `row` sees, from the first on.
__device__ __forceinline__ int kv_limit(const AttendArgs& a, KvSeq s, int row) {
  const int i = (uint32_t)row / (uint32_t)a.G;
  return i >= s.n ? 0 : a.causal ? kv_seen(s, i) : s.len;
}
// How many keys the rows [r0, r1) of a tile see, and how many of them one split takes (a multiple of `unit`).
__device__ __forceinline__ int kv_end(const AttendArgs& a, KvSeq s, int r0, int r1) {
  const int i1 = min((int)((uint32_t)(min(r1, a.R) - 1) / (uint32_t)a.G), s.n - 1);
  return (int)((uint32_t)r0 / (uint32_t)a.G) >= s.n ? 0 : a.causal ? kv_seen(s, i1) : s.len;
}
__device__ __forceinline__ int kv_chunk(const AttendArgs& a, int end, int unit) {
  return ((end + a.splits - 1) / a.splits + unit - 1) / unit * unit;
}

// ---- codes -----------------------------------------------------------------------------
__device__ __forceinline__ v8h codes_f16(uint32_t a, uint32_t b) {
  const v2h p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a, 1.0f, false);
  const v2h q = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a, 1.0f, true);
  const v2h r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, 1.0f, false);
  const v2h s = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, 1.0f, true);
  return v8h{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}
// Four words of four bytes -> word i holds byte i of each.
__device__ __forceinline__ void transpose4(const uint32_t (&k)[4], uint32_t (&o)[4]) {
  const uint32_t t0 = __builtin_amdgcn_perm(k[1], k[0], 0x05010400), t1 = __builtin_amdgcn_perm(k[1], k[0], 0x07030602);
  const uint32_t u0 = __builtin_amdgcn_perm(k[3], k[2], 0x05010400), u1 = __builtin_amdgcn_perm(k[3], k[2], 0x07030602);
  o[0] = __builtin_amdgcn_perm(u0, t0, 0x05040100), o[1] = __builtin_amdgcn_perm(u0, t0, 0x07060302);
  o[2] = __builtin_amdgcn_perm(u1, t1, 0x05040100), o[3] = __builtin_amdgcn_perm(u1, t1, 0x07060302);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) { return cvt_pk_16<MXF8_F16>(a, b); }

// Max / sum over the lanes that hold one row: LANES 16 (four of them, lanes l + 16 i) or 32 (lanes l, l + 32).
template <int LANES, class F>
__device__ __forceinline__ float row_reduce(float v, F f) {
  if constexpr (LANES == 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
// m for a largest x + e of `top`.  (Beside scores of 2^20 KV_UP would be rounded, up to 16 where their steps are 16.)
__device__ __forceinline__ float up_of(float top) { return top - (fabsf(top) < 0x1p20f ? KV_UP : 0.0f); }
__device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float sum_of(float a, float b) { return a + b; }

// Eight channels of a query to fp16, and the largest of their sizes, for bf16 (bits).
template <int DT>
__device__ __forceinline__ v8h query_f16(const Raw8<DT>& r, float s) {
  if constexpr (DT == MXF8_F16) {
    return __builtin_bit_cast(v8h, v4i{(int)r.w[0], (int)r.w[1], (int)r.w[2], (int)r.w[3]});
  } else {
    float f[8];
    r.get(f);
    return __builtin_bit_cast(v8h, v4i{(int)pack_f16(f[0] * s, f[1] * s), (int)pack_f16(f[2] * s, f[3] * s),
                                       (int)pack_f16(f[4] * s, f[5] * s), (int)pack_f16(f[6] * s, f[7] * s)});
  }
}

// One row's fragments of a query: N pieces of eight channels at channel(i).
template <int DT, int N, class F>
__device__ __forceinline__ void load_query(const AttendArgs& a, int b, int hk, int row, Raw8<DT> (&r)[N], F channel) {
  const int i = (uint32_t)row / (uint32_t)a.G, g = row - i * a.G;
  const int64_t at = b * a.qs[0] + (hk * a.G + g) * a.qs[1] + i * a.qs[2];
#pragma unroll
  for (int j = 0; j < N; ++j) r[j].load(a.q, at + channel(j));
}
// The same as fp16 (zeros for a row that is not there), and the factor of its scores.
template <int DT, int LANES, int N>
__device__ __forceinline__ float scale_query(const AttendArgs& a, bool there, Raw8<DT> (&r)[N], v8h (&f)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (!there) r[j].zero();
  int e = 0;
  if constexpr (DT == MXF8_BF16) {
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float x[8];
      r[j].get(x);
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(x[k]));
    }
    top = row_reduce<LANES>(top, max_of);
    e = min(max((int)(__float_as_uint(top) >> 23) - 127, -126), 126);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    f[j] = query_f16<DT>(r[j], __uint_as_float((uint32_t)(127 - e) << 23));
    if (a.scale < 0.0f) f[j] = -f[j];  // so that the factor of the scores is not negative, and their largest its own
  }
  // (at least 2^-117: times a page's 2^-32 or more it is still no 0, which would make NaN of a score that is hidden as -inf;
  // scores under so small a factor, of products below 2^32 and pages up to 2^63, are below 2^-22)
  return fmaxf(fabsf(a.scale) * __uint_as_float((uint32_t)(127 + e) << 23), 0x1p-117f);
}
// The factor of a page's scores.  (Never infinite: products of 0 have a score of 0.)
__device__ __forceinline__ float page_factor(float factor, float scale) { return fminf(factor * scale, KV_LARGEST); }

// N consecutive channels of an output row.
template <int DT, int N>
__device__ __forceinline__ void store_row(void* base, int64_t i, const float (&f)[N]) {
  typedef uint32_t words __attribute__((ext_vector_type(N / 2), aligned(2)));
  words w;
#pragma unroll
  for (int j = 0; j < N / 2; ++j) w[j] = cvt_pk_16<DT>(f[2 * j], f[2 * j + 1]);
  *reinterpret_cast<words*>(static_cast<uint16_t*>(base) + i) = w;
}
__device__ __forceinline__ int64_t out_row(const AttendArgs& a, int b, int hk, int row) {
  const int i = (uint32_t)row / (uint32_t)a.G, g = row - i * a.G;
  return b * a.os[0] + (hk * a.G + g) * a.os[1] + i * a.os[2];
}

// ---- few rows --------------------------------------------------------------------------
// Up to 64 rows a key head (its G heads' S queries): a workgroup takes a part of the keys, its four waves every fourth
// step of 32 keys each, straight from memory into the layout of 16 x 16 x 32 products, and joins their sums at the end.
// No LDS on the way: a lane loads 16 channels of its key, and for the values 8 keys' D / 16 channels, which it transposes in
// registers.  The next steps' loads are in flight while a step is computed.
//
// Bound by memory where the parts are long: 8 key heads x 131149 keys x 128, one query of 32 heads, 268 MB in 43 us (6.2
// TB/s, a part from the last cache); 64 sequences of 129 to 8192 tokens 104 us (5.2), of 4600 each 110 (5.5).  Short parts are bound by
// the chain of lengths, page entries, codes and join, some 4 us, and by a lone wave's issue (a step of D = 128 takes
// it 0.8 us).  Three or four steps ahead are no faster, with fewer waves; more than two workgroups a compute unit only
// even out lengths.
//
// Against the kernel for many rows, 8 key heads, us here / there with the joins:
//   rows                            17           32           33           48           64
//   D = 64, 16 x 4096 keys          20.5 / 46.5  21.4 / 47.0  27.0 / 48.9  27.8 / 49.5  29.3 / 50.5
//   D = 64, 64 x 4096               56 / 166     61 / 171     91 / 178     94 / 182     101 / 184
//   D = 64, 1 x 32768               14.3 / 27.3  15.4 / 27.6  19.7 / 28.8  20.6 / 29.2  21.5 / 29.2
//   D = 128, 16 x 4096              29.7 / 53.0  31.4 / 53.5  53.9 / 55.9  54.7 / 57.1  57.0 / 58.2
//   D = 128, 64 x 4096              110 / 187    116 / 189    208 / 193    210 / 195    219 / 195
//   D = 128, 1 x 32768              20.5 / 31.7  21.3 / 32.1  38.4 / 33.3  39.3 / 34.1  41.5 / 35.0
// (33 rows of 128 channels and more hold one wave a SIMD: from 4% faster to 19% slower there.)
constexpr int FEW_ROWS = 64, FEW_UNIT = 128;

template <int D>
struct FewStep {
  v4i k[2][D / 64];
  uint32_t v[8][D / 64];
  bool there[2];
  uint32_t ks[2], vs[2];
};

template <int DT, int D, int NR>
__global__ __launch_bounds__(256, (D == 64 ? (NR == 1 ? 4 : NR == 2 ? 3 : 2) : NR == 1 ? 3 : 4 / NR)) void kv_attend_few_kernel(const AttendArgs a) {
  constexpr int KK = D / 32, DI = D / 16, W = D / 64, STEPS = D == 128 || NR > 1 ? 2 : 3;
  __shared__ float om[4][16][D + 4];
  __shared__ float ml[4][2][16 * NR];
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int split = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  // (before it is known which rows are there: the loads need not wait for the lengths)
  Raw8<DT> raw[NR][KK];
#pragma unroll
  for (int t = 0; t < NR; ++t)
    load_query(a, b, hk, min(16 * t + c, a.R - 1), raw[t], [&](int j) { return 64 * (j / 2) + 16 * q + 8 * (j % 2); });
  const KvSeq seq = kv_seq(a, b);
  const int end = kv_end(a, seq, 0, a.R), chunk = kv_chunk(a, end, FEW_UNIT);
  const int k0 = split * chunk, k1 = min(k0 + chunk, end);
  if (a.splits > 1 && k0 >= k1) return;

  v8h qf[NR][KK];
  float factor[NR];
  int limit[NR], low = INT32_MAX;
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    const int row = 16 * t + c;
    limit[t] = row < a.R ? kv_limit(a, seq, row) : 0;
    low = min(low, row < a.R ? limit[t] : INT32_MAX);
  }
#pragma unroll
  for (int off = 8; off; off >>= 1) low = min(low, __shfl_xor(low, off, 64));
  low = __builtin_amdgcn_readfirstlane(low);  // every row sees the keys before it

  float m[NR], l[NR];
  v4f o[NR][DI];
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    m[t] = KV_NONE, l[t] = 0.0f;
#pragma unroll
    for (int i = 0; i < DI; ++i) o[t][i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const int mask = (1 << a.c.shift) - 1;
  const uint32_t k_lane = c * D + 16 * q, v_lane = 4 * q * D + c * DI;
  auto pages = [&](int key0, int (&entry)[2]) {  // (behind the end: the last again)
#pragma unroll
    for (int g = 0; g < 2; ++g) entry[g] = kv_entry(a.c, b, min(key0 + 16 * g, k1 - 1) >> a.c.shift);
  };
  auto load = [&](int key0, const int (&entry)[2], FewStep<D>& s) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      // (no page: page 0 is read and not used)
      s.there[g] = key0 + 16 * g < k1 && kv_valid(a.c, entry[g]);
      const int64_t ph = (int64_t)(s.there[g] ? entry[g] : 0) * a.c.H + hk;
      const int64_t at = ((ph << a.c.shift) + ((key0 + 16 * g) & mask)) * D;
      s.ks[g] = a.c.ks[ph], s.vs[g] = a.c.vs[ph];
      // (addresses: a base that the wave shares and 32 bits of a lane's own)
      const gbytes k = (gbytes)(a.c.k + at), v = (gbytes)(a.c.v + at);
#pragma unroll
      for (int j = 0; j < W; ++j) s.k[g][j] = *(const __attribute__((address_space(1))) v4i*)(k + (k_lane + 64 * j));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if constexpr (W == 2) {
          const v2i x = *(const __attribute__((address_space(1))) v2i*)(v + (v_lane + j * D));
          s.v[4 * g + j][0] = x[0], s.v[4 * g + j][W - 1] = x[1];
        } else {
          s.v[4 * g + j][0] = *(const __attribute__((address_space(1))) uint32_t*)(v + (v_lane + j * D));
        }
    }
  };
  auto compute = [&](int key0, FewStep<D>& s) {
    const bool whole = key0 + 32 <= low && s.there[0] && s.there[1];
    float ks[2], ev[2], iv[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const uint32_t kb = !s.there[g] ? 127 : __builtin_amdgcn_readfirstlane(s.ks[g]);
      const uint32_t vb = !s.there[g] ? 127 : __builtin_amdgcn_readfirstlane(s.vs[g]);
      ks[g] = kv_scale(kb);
      const int e = (int)vb - 127;
      ev[g] = (float)e, iv[g] = __uint_as_float((uint32_t)(127 - e) << 23);
    }
    v8h pf[NR];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      v4f x[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              codes_f16((uint32_t)s.k[g][kk / 2][2 * (kk % 2)], (uint32_t)s.k[g][kk / 2][2 * (kk % 2) + 1]), qf[t][kk], acc,
              0, 0, 0);
        const float f = page_factor(factor[t], ks[g]);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[g][r] = __builtin_fmaf(acc[r], f, ev[g]);
      }
      if (!whole) {
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            x[g][r] = key0 + 16 * g + 4 * q + r < limit[t] && s.there[g] ? x[g][r] : -INFINITY;
      }
      const float top = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])),
                              fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
      if (__ballot(top - m[t] > KV_UP + KV_SLACK)) {
        const float next = fmaxf(m[t], up_of(row_reduce<16>(top, max_of))), alpha = __builtin_amdgcn_exp2f(m[t] - next);
        m[t] = next;
        l[t] *= alpha;
#pragma unroll
        for (int i = 0; i < DI; ++i) o[t][i] *= alpha;
      }
      float p[2][4];
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) p[g][r] = __builtin_amdgcn_exp2f(x[g][r] - m[t]);
#pragma unroll
      for (int g = 0; g < 2; ++g) l[t] = __builtin_fmaf((p[g][0] + p[g][1]) + (p[g][2] + p[g][3]), iv[g], l[t]);
      pf[t] = __builtin_bit_cast(v8h, v4i{(int)pack_f16(p[0][0], p[0][1]), (int)pack_f16(p[0][2], p[0][3]),
                                          (int)pack_f16(p[1][0], p[1][1]), (int)pack_f16(p[1][2], p[1][3])});
    }
    if (!whole) {  // what is not there may be NaN, which 0 does not cancel
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (key0 + 16 * g + 4 * q + r >= k1 || !s.there[g])
#pragma unroll
            for (int d = 0; d < W; ++d) s.v[4 * g + r][d] = 0;
    }
#pragma unroll
    for (int d = 0; d < W; ++d) {
      const uint32_t lo[4] = {s.v[0][d], s.v[1][d], s.v[2][d], s.v[3][d]};
      const uint32_t hi[4] = {s.v[4][d], s.v[5][d], s.v[6][d], s.v[7][d]};
      uint32_t tl[4], th[4];
      transpose4(lo, tl);
      transpose4(hi, th);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v8h vf = codes_f16(tl[i], th[i]);
#pragma unroll
        for (int t = 0; t < NR; ++t) o[t][4 * d + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[t], o[t][4 * d + i], 0, 0, 0);
      }
    }
  };

  // STEPS - 1 steps' loads are in flight while one is computed, and the page entries of one more
  int key = k0 + 32 * w;
  if (key < k1) {
    FewStep<D> s[STEPS];
    int entry[2];
    pages(key, entry);
#pragma unroll
    for (int u = 0; u + 1 < STEPS; ++u) {
      if (key + u * FEW_UNIT < k1) load(key + u * FEW_UNIT, entry, s[u]);
      pages(key + (u + 1) * FEW_UNIT, entry);
    }
#pragma unroll
    for (int t = 0; t < NR; ++t) factor[t] = scale_query<DT, 16>(a, limit[t] > 0, raw[t], qf[t]);
    for (;;) {
#pragma unroll
      for (int u = 0; u < STEPS; ++u) {
        const int next = key + (STEPS - 1) * FEW_UNIT;
        if (next < k1) load(next, entry, s[(u + STEPS - 1) % STEPS]);
        pages(next + FEW_UNIT, entry);
        compute(key, s[u]);
        key += FEW_UNIT;
        if (key >= k1) goto done;
      }
    }
  }
done:
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    l[t] = row_reduce<16>(l[t], sum_of);
    if (q == 0) ml[w][0][16 * t + c] = m[t], ml[w][1][16 * t + c] = l[t];
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    const int rt = 16 * t + c;
    const float top = fmaxf(fmaxf(ml[0][0][rt], ml[1][0][rt]), fmaxf(ml[2][0][rt], ml[3][0][rt]));
    const float f = __builtin_amdgcn_exp2f(m[t] - top);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < DI; i += 4)  // channel DI (4 q + r) + i
        *reinterpret_cast<v4f*>(&om[w][c][DI * (4 * q + r) + i]) =
            v4f{o[t][i][r] * f, o[t][i + 1][r] * f, o[t][i + 2][r] * f, o[t][i + 3][r] * f};
    __syncthreads();
    const int rr = threadIdx.x >> 4, row = 16 * t + rr, ch = (threadIdx.x & 15) * DI;
    if (row < a.R) {
      float sum[DI], mm[4], ll = 0.0f;
#pragma unroll
      for (int i = 0; i < DI; ++i) sum[i] = (om[0][rr][ch + i] + om[1][rr][ch + i]) + (om[2][rr][ch + i] + om[3][rr][ch + i]);
#pragma unroll
      for (int u = 0; u < 4; ++u) mm[u] = ml[u][0][row];
      const float top4 = fmaxf(fmaxf(mm[0], mm[1]), fmaxf(mm[2], mm[3]));
#pragma unroll
      for (int u = 0; u < 4; ++u) ll = __builtin_fmaf(ml[u][1][row], __builtin_amdgcn_exp2f(mm[u] - top4), ll);
      if (a.splits == 1) {
        const float inv = ll == 0.0f ? 0.0f : __fdiv_rn(1.0f, ll);
#pragma unroll
        for (int i = 0; i < DI; ++i) sum[i] *= inv;
        store_row<DT, DI>(a.o, out_row(a, b, hk, row) + ch, sum);
      } else {
        const int64_t at = (((int64_t)b * a.c.H + hk) * a.splits + split) * a.R + row;
#pragma unroll
        for (int i = 0; i < DI; i += 4)
          *reinterpret_cast<v4f*>(a.part + at * D + ch + i) = v4f{sum[i], sum[i + 1], sum[i + 2], sum[i + 3]};
        if (ch == 0) *reinterpret_cast<v2f*>(a.stat + at * 2) = v2f{top4, ll};
      }
    }
    if (t + 1 < NR) __syncthreads();
  }
}

// ---- many rows -------------------------------------------------------------------------
// A workgroup of eight waves takes 256 rows of a key head, 32 a wave, and goes through its keys in tiles of 64.  A tile's
// codes go into LDS once, the keys as they are, the values transposed and converted to fp16; a wave converts the keys'
// fragments as it reads them.
// The two waves of a SIMD (of the groups w < 4 and w >= 4) take turns with the matrix unit: between two barriers, group 0
// first makes the scores of its next tile and the value product of this one and then takes the next one's exponentials, group
// 1 first takes exponentials and then multiplies.  Fragments are read from LDS well before their products, and each wave
// stages its share of the keys of tile j + 3 and the values of j + 1 among them.
//
// A tile's 2048 cycles of products take some 4000 (over the whole launch the matrix unit is 45% busy, the vector unit 56%, LDS
// 40%), at a clock under the power limit: 1.8-2.0 of 2.4 GHz.  1560 queries x 24 heads of 128 over 21840 keys: 457-476 us with the join's 18, 880-915 TFLOP/s
// (a library product of 8192^3 in fp16 reaches 1147 here).  What the parts bring there: both groups in the same order 492, without
// the wave priorities 470, a barrier between the two phases as well 518, key codes converted at each read instead of once
// 517, fragments read as they are needed 560-590.  One wave a SIMD with 64 rows and 512 registers would read LDS half as often,
// but the compiler then keeps the scores in accumulation registers and spills.
constexpr int MANY_ROWS = 256, MANY_KEYS = 64;

// LDS, in 16-byte chunks with a swizzle: keys [64][D] and values [D][64] in fp16; of each granule of 16 keys, the keys'
// scale, the values' exponent and 2^-that, and whether it is there.
template <int D>
struct ManyLds {
  v4i k[4][MANY_KEYS * D / 8];
  v4i v[2][D * MANY_KEYS / 8];
  v4f scale[4][4];
  v4f unused[64];  // where the other lanes of a wave write when one writes a scale
};
template <int D>
__device__ __forceinline__ int many_k(int key, int chunk) { return key * (D / 8) + (chunk ^ lds_swz<2 * D>(key)); }
__device__ __forceinline__ int many_v(int ch, int chunk) { return ch * 8 + (chunk ^ ((ch >> 1 ^ ch >> 4) & 7)); }

template <int DT, int D>
__global__ __launch_bounds__(512, 2) void kv_attend_many_kernel(const AttendArgs a) {
  constexpr int KK = D / 16, OT = D / 32;  // products a score tile; output tiles
  __shared__ ManyLds<D> lds;
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = w >> 2;
  // Neighbouring workgroups take different key heads: where their number is a multiple of eight, all that read one head's keys
  // are on one XCD, and its L2 has them.  The last rows come first: under a causal mask they see the most keys.
  const int groups = a.c.H * a.B, x0 = blockIdx.x / groups, hb = blockIdx.x % groups;
  const int tiles = (a.R + MANY_ROWS - 1) / MANY_ROWS, split = x0 / tiles, r0 = (tiles - 1 - x0 % tiles) * MANY_ROWS;
  const int hk = hb % a.c.H, b = hb / a.c.H;
  const int row = r0 + 32 * w + c;
  Raw8<DT> raw[KK];
  load_query(a, b, hk, min(row, a.R - 1), raw, [&](int j) { return 16 * j + 8 * h; });
  const KvSeq seq = kv_seq(a, b);
  const int end = kv_end(a, seq, r0, r0 + MANY_ROWS), chunk = kv_chunk(a, end, MANY_KEYS);
  const int k0 = split * chunk, k1 = min(k0 + chunk, end);
  if (a.splits > 1 && k0 >= k1) return;

  const int limit = row < a.R ? kv_limit(a, seq, row) : 0;
  int low = row < a.R ? limit : INT32_MAX, high = limit;
  v8h qf[KK];
  const float factor = scale_query<DT, 32>(a, limit > 0, raw, qf);
  // One fma makes a probability's exponent, whose product is unrounded and whose sum e - m is not: with scores of 2^20 it is off
  // by up to 2^-3, with larger ones it would leave fp16's range.  A wave that has such rows, or rows whose factor
  // may overflow, rounds the scores first, as their maximum was.
  bool far = __ballot(factor >= 0x1p64f) != 0;
  float m = KV_NONE, l = 0.0f;
  v16f o[OT];
#pragma unroll
  for (int i = 0; i < OT; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.0f;
#pragma unroll
  for (int off = 16; off; off >>= 1) low = min(low, __shfl_xor(low, off, 64)), high = max(high, __shfl_xor(high, off, 64));
  // every row of the wave sees the keys before `low`, none those from `high` on
  low = __builtin_amdgcn_readfirstlane(low), high = __builtin_amdgcn_readfirstlane(high);

  // Each wave stages 16 bytes a lane of one granule of 16 keys.  D = 128: half of granule w / 2, 8 of its keys and two times
  // 4 of its values' keys; D = 64: waves 0 to 3 the keys of granule w, waves 4 to 7 the values of granule w - 4.
  const int mask = (1 << a.c.shift) - 1;
  const int gran = D == 128 ? w >> 1 : w & 3;
  const bool has_k = D == 128 || w < 4, has_v = D == 128 || w >= 4;
  const int skey = D == 128 ? (w & 1) * 8 + (lane >> 3) : lane >> 2, sch = D == 128 ? lane & 7 : lane & 3;
  const int vu = D == 128 ? (w & 1) * 2 + (lane >> 5) : lane >> 4, vch = lane % (D / 4) * 4;  // values 4 vu + j, 4 channels
  v4i kreg;
  uint32_t vreg[4], ksb = 127, vsb = 127;
  bool kthere = false, vthere = false;
  auto index = [&](int j) { return min(k0 + j * MANY_KEYS + 16 * gran, k1 - 1) >> a.c.shift; };  // (behind the end: the last)
  auto entry = [&](int j) { return kv_entry(a.c, b, index(j)); };
  // (the same as a vector load: a scalar one would make every wait for LDS a wait for it)
  const int zero = __builtin_amdgcn_mbcnt_lo(0, 0);
  auto entry_ahead = [&](int j) { return a.c.table[b * a.c.table_stride + index(j) + zero]; };
  auto place = [&](int j, int page, bool& there) {  // (no page: page 0 is read and not used)
    there = k0 + j * MANY_KEYS + 16 * gran < k1 && kv_valid(a.c, page);
    return (int64_t)(there ? page : 0) * a.c.H + hk;
  };
  auto load_k = [&](int j, int page) {  // of tile j of this split
    if (!has_k) return;
    const int64_t ph = place(j, page, kthere);
    const uint8_t* p = a.c.k + ((ph << a.c.shift) + ((k0 + j * MANY_KEYS + 16 * gran) & mask)) * D;
    kreg = *reinterpret_cast<const v4i*>(p + skey * D + 16 * sch);
    ksb = a.c.ks[ph], vsb = a.c.vs[ph];
  };
  auto load_v = [&](int j, int page) {
    if (!has_v) return;
    const int64_t ph = place(j, page, vthere);
    const uint8_t* p = a.c.v + ((ph << a.c.shift) + ((k0 + j * MANY_KEYS + 16 * gran) & mask)) * D;
#pragma unroll
    for (int i = 0; i < 4; ++i) vreg[i] = *reinterpret_cast<const uint32_t*>(p + (4 * vu + i) * D + vch);
  };
  const int put_k_at[2] = {many_k<D>(16 * gran + skey, 2 * sch), many_k<D>(16 * gran + skey, 2 * sch + 1)};
  int put_v_at[4];  // in halves of chunks
#pragma unroll
  for (int i = 0; i < 4; ++i) put_v_at[i] = 2 * many_v(vch + i, 2 * gran + (vu & 1)) + (vu >> 1);
  v4f* const scale_at = skey == 0 && sch == 0 ? &lds.scale[0][gran] : &lds.unused[lane];
  auto put_k = [&](int j) {
    if (!has_k) return;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      lds.k[j & 3][put_k_at[i]] = __builtin_bit_cast(v4i, codes_f16((uint32_t)kreg[2 * i], (uint32_t)kreg[2 * i + 1]));
    const uint32_t kb = kthere ? ksb : 127, vb = kthere ? vsb : 127;
    scale_at[skey == 0 && sch == 0 ? (j & 3) * 4 : 0] =
        v4f{kv_scale(kb), (float)((int)vb - 127), __uint_as_float((254 - vb) << 23), kthere ? 1.0f : 0.0f};
  };
  auto put_v = [&](int j) {
    if (!has_v) return;
    // what is not there may be NaN, which a probability of 0 does not cancel
    const int there = vthere ? k1 - (k0 + j * MANY_KEYS + 16 * gran + 4 * vu) : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) vreg[i] = i < there ? vreg[i] : 0;
    // keys 16 t + 4 h + 0 .. 3 and 16 t + 8 + 4 h + 0 .. 3 are the chunk that half h of a wave reads for step t
    uint32_t x[4];
    transpose4(vreg, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const v2h lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)x[i], 1.0f, false);
      const v2h hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)x[i], 1.0f, true);
      reinterpret_cast<v2i*>(lds.v[j & 1])[put_v_at[i]] = v2i{__builtin_bit_cast(int, lo), __builtin_bit_cast(int, hi)};
    }
  };

  int kat[KK], vat[4];  // chunks of this lane's fragments in a buffer
#pragma unroll
  for (int i = 0; i < KK; ++i) kat[i] = many_k<D>(c, 2 * i + h);
#pragma unroll
  for (int g = 0; g < 4; ++g) vat[g] = many_v(c, 2 * g + h);  // channel 32 i + c, chunk 2 g + h: vat[g ^ i], 256 i further

  v16f x[2];
  v8h pf[4];
  v4i kf[KK][2], vf[4][OT];
  auto read_k = [&](int j, int part) {  // half of a tile's fragments, by channels
#pragma unroll
    for (int i = part * KK / 2; i < (part + 1) * KK / 2; ++i)
#pragma unroll
      for (int g = 0; g < 2; ++g) kf[i][g] = lds.k[j & 3][kat[i] + g * 32 * (D / 8)];
  };
  auto read_v = [&](int j, int g) {
#pragma unroll
    for (int i = 0; i < OT; ++i) vf[g][i] = lds.v[j & 1][vat[g ^ i] + 256 * i];
  };
  auto scores = [&](int part) {
    if (part == 0) {
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[g][r] = 0.0f;
    }
#pragma unroll
    for (int i = part * KK / 2; i < (part + 1) * KK / 2; ++i)
#pragma unroll
      for (int g = 0; g < 2; ++g) x[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, kf[i][g]), qf[i], x[g], 0, 0, 0);
  };
  auto values = [&](int g) {
#pragma unroll
    for (int i = 0; i < OT; ++i)
      o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, vf[g][i]), pf[g], o[i], 0, 0, 0);
  };
  auto exponentials = [&](int j) {
    const int key0 = k0 + j * MANY_KEYS;
    float f[4], e[4], iv[4], n[4], y[4];
    v4f s[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) s[g] = lds.scale[j & 3][g];
    auto tops = [&]() {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        y[g] = x[g >> 1][(g & 1) * 8];
#pragma unroll
        for (int r = 1; r < 8; ++r) y[g] = fmaxf(y[g], x[g >> 1][(g & 1) * 8 + r]);
      }
    };
    tops();
    bool all = key0 + MANY_KEYS <= low;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f[g] = factor * s[g][0], e[g] = s[g][1], iv[g] = s[g][2];
      all = all & (__builtin_amdgcn_readfirstlane(__float_as_uint(s[g][3])) != 0);
    }
    if (far) {
#pragma unroll
      for (int g = 0; g < 4; ++g) f[g] = page_factor(factor, s[g][0]);
    }
    if (!all) {
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int r = 0; r < 8; ++r)
          x[g >> 1][(g & 1) * 8 + r] = key0 + 16 * g + 8 * (r >> 2) + 4 * h + (r & 3) < limit && s[g][3] != 0.0f
                                           ? x[g >> 1][(g & 1) * 8 + r]
                                           : -INFINITY;
      tops();
    }
    float top = -INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g) top = fmaxf(top, __builtin_fmaf(y[g], f[g], e[g]));
    if (__ballot(top - m > KV_UP + KV_SLACK)) {
      const float next = fmaxf(m, up_of(row_reduce<32>(top, max_of))), alpha = __builtin_amdgcn_exp2f(m - next);
      m = next;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < OT; ++i) o[i] *= alpha;
      far |= __ballot(fabsf(m) >= 0x1p20f && m != KV_NONE) != 0;
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) n[g] = e[g] - m;
    if (far) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
#pragma unroll
        for (int r = 0; r < 8; ++r)
          x[g >> 1][(g & 1) * 8 + r] = __builtin_fmaf(x[g >> 1][(g & 1) * 8 + r], f[g], e[g]) - m;
        f[g] = 1.0f, n[g] = 0.0f;
      }
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float sum = 0.0f;
      v4i words;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[g >> 1][(g & 1) * 8 + 2 * r], f[g], n[g]));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[g >> 1][(g & 1) * 8 + 2 * r + 1], f[g], n[g]));
        words[r] = (int)pack_f16(p0, p1);
        sum += p0 + p1;
      }
      l = __builtin_fmaf(sum, iv[g], l);
      pf[g] = __builtin_bit_cast(v8h, words);
    }
  };
  // (a phase's products and exponentials stay in it)
  auto change = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
  };

  const int n = (k1 - k0 + MANY_KEYS - 1) / MANY_KEYS;  // tiles
  if (n > 0) {
    int page[3] = {entry(0), entry(1), entry(2)};
    load_v(0, page[0]);
    v4i first_k[3];
    uint32_t first_s[3][2];
    bool first_there[3];
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      load_k(j, page[j]);
      first_k[j] = kreg, first_s[j][0] = ksb, first_s[j][1] = vsb, first_there[j] = kthere;
    }
    put_v(0);
    load_v(1, page[1]);
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      kreg = first_k[j], ksb = first_s[j][0], vsb = first_s[j][1], kthere = first_there[j];
      put_k(j);
    }
    page[0] = page[2], page[1] = entry(3), page[2] = entry(4);  // of tiles j + 2, j + 3, j + 4
    load_k(3, page[1]);
    int ahead = entry_ahead(5);
    change();
    read_k(0, 0);
    read_k(0, 1);
    scores(0);
    scores(1);
    auto fetch = [&](int j) {
      load_v(j + 2, page[0]);
      load_k(j + 4, page[2]);
      page[0] = page[1], page[1] = page[2], page[2] = __builtin_amdgcn_readfirstlane(ahead);
      ahead = entry_ahead(j + 6);
    };
    // a wave whose rows see nothing of a tile, or that has none, only stages
    auto sees = [&](int j) { return k0 + j * MANY_KEYS < high; };
    if (!group && sees(0)) exponentials(0);
    read_k(1, 0);
    for (int j = 0; j + 1 < n; ++j) {
      if (sees(j)) {
        if (group) exponentials(j);
        __builtin_amdgcn_s_setprio(1);
        read_k(j + 1, 1);
        scores(0);
        put_k(j + 3);
        __builtin_amdgcn_sched_barrier(0);
        read_v(j, 0);
        read_v(j, 1);
        scores(1);
        put_v(j + 1);
        __builtin_amdgcn_sched_barrier(0);
        read_v(j, 2);
        read_v(j, 3);
        values(0);
        values(1);
        fetch(j);
        values(2);
        values(3);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        if (!group) exponentials(j + 1);
        read_k(j + 2, 0);
      } else {
        put_k(j + 3);
        put_v(j + 1);
        fetch(j);
      }
      change();
    }
    if (sees(n - 1)) {
      if (group) exponentials(n - 1);
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (g == 0 || k0 + (n - 1) * MANY_KEYS + 16 * g < k1) {
          read_v(n - 1, g);
          values(g);
        }
    }
  }
  l = row_reduce<32>(l, sum_of);
  if (a.splits == 1) {
    // rows of the output through LDS, where this wave's keys were, so that a row is stored at once
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    __syncthreads();
    v2i* mine = reinterpret_cast<v2i*>(lds.k) + w * 32 * (D / 4);
    auto at = [&](int r, int piece) { return r * (D / 4) + (piece ^ (r & 15)); };  // pieces of four channels
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        mine[at(c, 8 * i + 2 * g + h)] = v2i{(int)cvt_pk_16<DT>(o[i][4 * g] * inv, o[i][4 * g + 1] * inv),
                                             (int)cvt_pk_16<DT>(o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv)};
    __builtin_amdgcn_wave_barrier();  // (LDS operations of a wave complete in order)
    constexpr int L = D / 8;          // lanes of a row
#pragma unroll
    for (int i = 0; i < 32 * L / 64; ++i) {
      const int r = i * (64 / L) + lane / L, to = r0 + 32 * w + r;
      const v2i u = mine[at(r, lane % L * 2)], v = mine[at(r, lane % L * 2 + 1)];
      if (to < a.R)
        *reinterpret_cast<words4*>(static_cast<uint16_t*>(a.o) + out_row(a, b, hk, to) + lane % L * 8) =
            words4{(uint32_t)u[0], (uint32_t)u[1], (uint32_t)v[0], (uint32_t)v[1]};
    }
  } else if (row < a.R) {
    const int64_t at = (((int64_t)b * a.c.H + hk) * a.splits + split) * a.R + row;
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<v4f*>(a.part + at * D + 32 * i + 8 * g + 4 * h) =
            v4f{o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]};
    if (h == 0) *reinterpret_cast<v2f*>(a.stat + at * 2) = v2f{m, l};
  }
}

// ---- splits joined ---------------------------------------------------------------------
constexpr int KV_MAX_SPLITS = 64;

// One row to WAVES waves: the splits' maxima and sums in a lane each, then their outputs, four channels a lane and 256 / D
// splits at once, U times in flight together.  The first loads do not wait to know how many splits there are.
template <int DT, int D, int WAVES, int U>
__global__ __launch_bounds__(256) void kv_attend_join_kernel(const AttendArgs a, int rows, int unit) {
  constexpr int L = D / 4, P = 64 / L;  // lanes of a split, splits at once
  __shared__ v4f sums[4][64];
  const int lane = threadIdx.x & 63, hk = blockIdx.y, b = blockIdx.z;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x * (4 / WAVES) + w / WAVES;
  if (WAVES == 1 && row >= a.R) return;
  const int64_t at = (((int64_t)b * a.c.H + hk) * a.splits) * a.R + row;
  const float* part = a.part + at * D + lane % L * 4;
  const int first = w % WAVES * P + lane / L;  // this lane's splits: first, first + P WAVES, ...
  auto load = [&](int s) { return *reinterpret_cast<const v4f*>(part + (int64_t)s * a.R * D); };
  v4f x[U];
#pragma unroll
  for (int i = 0; i < U; ++i) x[i] = load(min(first + i * P * WAVES, a.splits - 1));
  float m = KV_NONE, l = 0.0f;
  const v2f st = *reinterpret_cast<const v2f*>(a.stat + (at + (int64_t)min(lane, a.splits - 1) * a.R) * 2);
  const int r0 = row / rows * rows, end = kv_end(a, kv_seq(a, b), r0, r0 + rows);
  const int chunk = kv_chunk(a, end, unit), n = end ? (end + chunk - 1) / chunk : 0;
  if (lane < n) m = st[0], l = st[1];
  const float f = __builtin_amdgcn_exp2f(m - lanes_max<64>(m));
  const float sum = lanes_sum<64>(l * f);
  v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = first;; s0 += U * P * WAVES) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int s = s0 + i * P * WAVES;
      const float fs = __shfl(f, s & 63, 64);
      if (s < n) o += x[i] * fs;
    }
    if (s0 - lane / L + U * P * WAVES >= n) break;
#pragma unroll
    for (int i = 0; i < U; ++i) x[i] = load(min(s0 + (U + i) * P * WAVES, a.splits - 1));
  }
#pragma unroll
  for (int off = L; off < 64; off *= 2)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], off, 64);
  if constexpr (WAVES > 1) {
    sums[w][lane] = o;
    __syncthreads();
    if (w % WAVES) return;
#pragma unroll
    for (int i = 1; i < WAVES; ++i) o += sums[w + i][lane];
  }
  if (lane >= L || row >= a.R) return;
  const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
  const float z[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  store_row<DT, 4>(a.o, out_row(a, b, hk, row) + lane * 4, z);
}

// ---- plan ------------------------------------------------------------------------------
struct AttendPlan {
  bool few;
  int splits;
  int64_t rows, tiles;  // rows a key head, row tiles of them
};
static AttendPlan plan_attend(int64_t B, int64_t H, int64_t Hk, int64_t S, int64_t D, int64_t width, int64_t page) {
  AttendPlan p{};
  p.rows = S * (H / Hk);
  p.few = p.rows <= FEW_ROWS;
  p.tiles = p.few ? 1 : cdiv(p.rows, MANY_ROWS);
  const int64_t groups = B * Hk * p.tiles, keys = width * page;
  p.splits = 1;
  if (p.few) {
    // Two workgroups a compute unit, however short their parts are; up to eight where each still has 1024 keys, which evens
    // out sequences of different lengths.  KV_MAX_SPLITS, as many as a wave of the join has lanes, ends both: one sequence's
    // 131072 keys of one head are read by 64 workgroups, 1.6 TB/s (22 us; of two heads 22, of four 26, of eight 45).
    const int64_t few = cdiv(512, groups), parts = cdiv(keys, FEW_UNIT), more = cdiv(2048, groups), thousands = keys / 1024;
    const int64_t n = more < thousands ? more : thousands, m = few < parts ? few : parts;
    p.splits = (int)(n > m ? n : m);
  } else {
    // The rounds that the workgroups make over the compute units, of so many tiles each and some three tiles' time to begin
    // and end, and joining: about five tiles' time, and two passes over the sums at 5 TB/s.
    double best = 0.0;
    for (int n = 1; n <= KV_MAX_SPLITS && (n == 1 || (n * 4 * MANY_KEYS <= keys && groups * n <= 2048)); ++n) {
      const double rounds = (double)cdiv(groups * n, 256), each = (double)cdiv(cdiv(keys, n), MANY_KEYS) + 3.0;
      const double join = n == 1 ? 0.0 : 5.0 + (double)groups * n * MANY_ROWS * D * 8.0 / 5.0e6;
      if (n == 1 || rounds * each + join < best) best = rounds * each + join, p.splits = n;
    }
  }
  if (p.splits > KV_MAX_SPLITS) p.splits = KV_MAX_SPLITS;
  if (p.splits < 1) p.splits = 1;
  return p;
}

template <int DT, int D>
static int launch_attend(AttendArgs& a, const AttendPlan& p, int B, hipStream_t st) {
  const char* what = "kv_attend";
  const int Hk = a.c.H;
  if (p.few) {
    const dim3 grid(p.splits, Hk, B);
    if (a.R <= 16)
      kv_attend_few_kernel<DT, D, 1><<<grid, 256, 0, st>>>(a);
    else if (a.R <= 32)
      kv_attend_few_kernel<DT, D, 2><<<grid, 256, 0, st>>>(a);
    else
      kv_attend_few_kernel<DT, D, 4><<<grid, 256, 0, st>>>(a);
  } else {
    const int64_t blocks = p.tiles * p.splits * Hk * B;
    if (!grid_fits(blocks, 512)) return set_error(MXF8_EINVAL, "%s: shape too large", what);
    kv_attend_many_kernel<DT, D><<<dim3((unsigned)blocks), 512, 0, st>>>(a);
  }
  if (const int rc = check_launch(what)) return rc;
  if (p.splits == 1) return MXF8_OK;
  const int rows = p.few ? FEW_ROWS : MANY_ROWS, unit = p.few ? FEW_UNIT : MANY_KEYS;
  if (p.splits > 16)  // (more than a wave reads at once, D = 128)
    kv_attend_join_kernel<DT, D, 4, 8><<<dim3((unsigned)a.R, Hk, B), 256, 0, st>>>(a, rows, unit);
  else if (p.splits > 4)
    kv_attend_join_kernel<DT, D, 1, 8><<<dim3((unsigned)cdiv(a.R, 4), Hk, B), 256, 0, st>>>(a, rows, unit);
  else
    kv_attend_join_kernel<DT, D, 1, 2><<<dim3((unsigned)cdiv(a.R, 4), Hk, B), 256, 0, st>>>(a, rows, unit);
  return check_launch(what);
}

}  // namespace mxf8

using namespace mxf8;

extern "C" int64_t mxf8_kv_attend_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t S, int64_t D,
                                                  int64_t table_width, int64_t page_size) {
  if (B <= 0 || H <= 0 || Hk <= 0 || H % Hk || S <= 0 || D <= 0 || table_width <= 0 || page_size <= 0) return 0;
  const AttendPlan p = plan_attend(B, H, Hk, S, D, table_width, page_size);
  return p.splits == 1 ? 0 : B * Hk * p.splits * p.rows * (D + 2) * 4;
}

extern "C" int mxf8_kv_attend(const void* q, const int64_t q_strides[4], int dtype, int64_t B, int64_t H, int64_t S,
                              int64_t D, const uint8_t* k_codes, const uint8_t* v_codes, const uint8_t* k_scale,
                              const uint8_t* v_scale, int64_t pages, int64_t Hk, int64_t page_size,
                              const int32_t* page_table, int64_t table_stride, int64_t table_width,
                              const int32_t* lengths, const int32_t* q_lengths, int causal, float scale, void* out,
                              const int64_t out_strides[4], void* workspace, hipStream_t stream) {
  const char* what = "kv_attend";
  AttendArgs a{};
  if (const int rc = kv_check_pages(what, k_codes, v_codes, k_scale, v_scale, pages, Hk, page_size, D, page_table,
                                    table_stride, table_width, B, &a.c))
    return rc;
  if (H < 0 || H > 65535 || S < 0) return set_error(MXF8_EINVAL, "%s: bad shape", what);
  if (H && (Hk == 0 || H % Hk))
    return set_error(MXF8_EINVAL, "%s: %lld heads over %lld key heads", what, (long long)H, (long long)Hk);
  if (dtype != MXF8_BF16 && dtype != MXF8_F16) return set_error(MXF8_EINVAL, "%s: bad dtype %d", what, dtype);
  if (!__builtin_isfinite(scale)) return set_error(MXF8_EINVAL, "%s: scale must be finite", what);
  if (B == 0 || H == 0 || S == 0) return MXF8_OK;
  if (!q || !out || !q_strides || !out_strides || !lengths) return set_error(MXF8_EINVAL, "%s: null pointer", what);
  if (q_strides[3] != 1 || out_strides[3] != 1)
    return set_error(MXF8_EINVAL, "%s: channels must be contiguous", what);
  if (S > (1 << 28) || S * (H / Hk) > (1 << 28)) return set_error(MXF8_EINVAL, "%s: shape too large", what);
  const AttendPlan p = plan_attend(B, H, Hk, S, D, table_width, page_size);
  if (p.splits > 1 && (!workspace || (uintptr_t)workspace % 16))
    return set_error(MXF8_EINVAL, "%s: a 16-byte aligned workspace is needed", what);
  if (pages == 0) a.c.width = 0;  // no keys
  a.q = q, a.o = out;
  for (int i = 0; i < 3; ++i) a.qs[i] = q_strides[i], a.os[i] = out_strides[i];
  a.lengths = lengths, a.q_lengths = q_lengths;
  a.B = (int)B, a.S = (int)S, a.G = (int)(H / Hk), a.R = (int)p.rows, a.causal = causal != 0;
  a.scale = scale * 1.4426950408889634f;
  a.splits = p.splits;
  a.part = static_cast<float*>(workspace);
  a.stat = a.part + B * Hk * p.splits * p.rows * D;
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return D == 128 ? launch_attend<DT, 128>(a, p, (int)B, stream) : launch_attend<DT, 64>(a, p, (int)B, stream);
  };
  return dtype == MXF8_BF16 ? launch(std::integral_constant<int, MXF8_BF16>{})
                            : launch(std::integral_constant<int, MXF8_F16>{});
}
