// Writing and reading a paged e4m3 cache of keys and values.
//
//   page p, head h holds 2^e and codes c with value = c 2^e, e the smallest exponent in [-32, 63] with
//   max |x| <= 448 2^e over its tokens; code = the nearest e4m3 number to x 2^-e, ties to even, 448 at most.
//   Tokens appended to a page that holds others raise its exponent where theirs is larger; what was held is then rounded
//   again, from its codes.  The exponent falls only when a page's first token is written again.
// A power of two costs a floating code nothing but range, makes that second rounding exact for all but the smallest
// values, and lets a reader apply it exactly.
#include <type_traits>

#include "kv_cache.h"
#include "rowio.h"

namespace mxf8 {

int kv_check_pages(const char* what, const void* k, const void* v, const void* ks, const void* vs, int64_t pages,
                   int64_t H, int64_t page, int64_t D, const int32_t* table, int64_t table_stride, int64_t width,
                   int64_t B, KvPages* c) {
  if (D != 64 && D != 128) return set_error(MXF8_EINVAL, "%s: D must be 64 or 128, got %lld", what, (long long)D);
  if (page != 16 && page != 32 && page != 64 && page != 128)
    return set_error(MXF8_EINVAL, "%s: a page holds 16, 32, 64 or 128 tokens, got %lld", what, (long long)page);
  if (pages < 0 || pages > INT32_MAX || H < 0 || H > 65535 || B < 0 || B > 65535 || width < 0 ||
      width > (1 << 30) / page)
    return set_error(MXF8_EINVAL, "%s: bad shape", what);
  if (width && B > 1 && table_stride < width)
    return set_error(MXF8_EINVAL, "%s: page table rows overlap", what);
  if (pages && H && (!k || !v || !ks || !vs)) return set_error(MXF8_EINVAL, "%s: null pointer", what);
  if (width && B && !table) return set_error(MXF8_EINVAL, "%s: null page table", what);
  if (((uintptr_t)k | (uintptr_t)v) % 16) return set_error(MXF8_EINVAL, "%s: codes must be 16-byte aligned", what);
  c->k = static_cast<const uint8_t*>(k), c->v = static_cast<const uint8_t*>(v);
  c->ks = static_cast<const uint8_t*>(ks), c->vs = static_cast<const uint8_t*>(vs);
  c->table = table, c->table_stride = table_stride, c->pages = pages;
  c->H = (int)H, c->width = (int)width, c->shift = __builtin_ctz((unsigned)page);
  return MXF8_OK;
}

// The smallest e in [KV_E_MIN, KV_E_MAX] with amax <= 448 2^e = 1.75 2^(e + 8), of a finite amax >= 0.
__device__ __forceinline__ int kv_exponent(float amax) {
  return min(max((int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 135, KV_E_MIN), KV_E_MAX);
}
__device__ __forceinline__ float kv_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// What happens to a key on the way: nothing; the norm or the rotation of neighbouring channels, or both; with half-split pairs,
// whose partners are at the same place of another lane's eight (P % 8 == 0), or anywhere.
enum { KEY_PLAIN, KEY_PAIRS, KEY_HALF, KEY_HALF_ANY };

struct AppendArgs {
  KvPages c;
  const void *x[2], *w;   // keys and values; the key norm's weight or null
  int64_t xs[2][3];       // strides of batch, head, token
  const float* turns;     // cos / sin [.., S, P, 2]
  int64_t turns_batch;
  const int32_t *starts, *counts;
  int S, P;
  int eights;  // groups of eight pages that go through their heads together
  float eps;
};

// f over the L (8 or 16) neighbouring lanes that hold a token.
template <int L>
__device__ __forceinline__ double lanes_sum64(double v) {
#define MXF8_STEP(CTRL)                                                                                            \
  {                                                                                                                \
    const uint64_t u = __builtin_bit_cast(uint64_t, v);                                                            \
    const uint32_t lo = __builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xf, 0xf, true);                          \
    const uint32_t hi = __builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);                  \
    v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);                                                      \
  }
  MXF8_STEP(0xb1)
  MXF8_STEP(0x4e)
  MXF8_STEP(0x141)
  if constexpr (L == 16) MXF8_STEP(0x140)
#undef MXF8_STEP
  return v;
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, off, 64));
  return v;
}

template <int N>
__device__ __forceinline__ uint32_t block_max(const uint32_t (&waves)[N]) {
  uint32_t v = waves[0];
#pragma unroll
  for (int i = 1; i < N; ++i) v = max(v, waves[i]);
  return v;
}

// The largest |x| of eight as stored: of 16 bits in both halves, of fp32 as it is; infinities and NaN come last.
template <int DT>
__device__ __forceinline__ uint32_t raw_max(const Raw8<DT>& r, uint32_t top) {
  if constexpr (DT == MXF8_F32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(r.w[j]) & 0x7fffffffu);
  } else {
    typedef unsigned short v2u __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < 4; ++j)
      top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(v2u, top),
                                                                   __builtin_bit_cast(v2u, r.w[j] & 0x7fff7fffu)));
  }
  return top;
}
// raw_max's result as fp32 bits
template <int DT>
__device__ __forceinline__ uint32_t raw_max_f32(uint32_t top) {
  if constexpr (DT == MXF8_F32) return top;
  const uint32_t t = max(top & 0xffffu, top >> 16);
  return DT == MXF8_BF16 ? t << 16 : __float_as_uint(f16_bits_to_f32(t));
}

// Eight values to codes under 2^e; none is larger than 448 2^e.
typedef short v2s __attribute__((ext_vector_type(2)));
__device__ __forceinline__ v2i codes_of(const float (&f)[8], float scale) {
  v2s w[2] = {};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    w[j] = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w[j], f[4 * j], f[4 * j + 1], scale, false);
    w[j] = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w[j], f[4 * j + 2], f[4 * j + 3], scale, true);
  }
  return v2i{__builtin_bit_cast(int, w[0]), __builtin_bit_cast(int, w[1])};
}
template <int DT>
__device__ __forceinline__ v2i codes_of(const Raw8<DT>& r, float scale) {
  if constexpr (DT == MXF8_F32) {
    float f[8];
    r.get(f);
    return codes_of(f, scale);
  } else {
    v2s w[2] = {};
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if constexpr (DT == MXF8_BF16) {
        w[j] = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w[j], __builtin_bit_cast(v2bf, r.w[2 * j]), scale, false);
        w[j] = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w[j], __builtin_bit_cast(v2bf, r.w[2 * j + 1]), scale, true);
      } else {
        w[j] = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w[j], __builtin_bit_cast(v2h, r.w[2 * j]), scale, false);
        w[j] = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w[j], __builtin_bit_cast(v2h, r.w[2 * j + 1]), scale, true);
      }
    return v2i{__builtin_bit_cast(int, w[0]), __builtin_bit_cast(int, w[1])};
  }
}

constexpr uint32_t INF_BITS = 0x7f800000u, LARGEST_BITS = 0x63600000u;  // of 448 2^63

// fp64 to fp32 on the way to a code: rounded to nearest, but off a border (of two codes, or of 448 2^e: a fp32 number whose last
// 19 bits are 0) that the value is not on.  So the code is the one nearest to the value in 64 bits.
__device__ __forceinline__ void round_keys(const double (&y)[8], float (&f)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float r = (float)y[j];
    const double d = y[j] - (double)r;
    const bool border = __float_as_uint(r) << 13 == 0 && r != 0.0f && fabsf(r) < INFINITY && d != 0.0;
    f[j] = border ? __uint_as_float(__float_as_uint(r) + ((d > 0.0) == (r > 0.0f) ? 1 : -1)) : r;
  }
}

// A workgroup writes one page and head of one sequence: D / 8 lanes hold a token's eight channels each, so the
// page's maximum is one reduction over values that stay in registers until they are rounded.  A key's code is the one that its
// norm and turn in fp64 give (fp32 would put two or three of a million on the wrong side of a border between two codes).  Keys of
// 16 bits are computed in fp32 whose error is known, and again in fp64 only by the waves, some 3% of them, that have a
// channel so near to a border that the error might decide; fp32 keys, and pairs that no lane holds whole, in fp64 alone.
//
// Bound by memory where keys stay as they are: 20280 tokens x 24 heads x 128 in bf16, 374 MB, 65 us (5.7 TB/s).  Normed and
// turned by neighbouring pairs 83 (the vector unit 59% busy; all in fp64 93 and 84%), half-split 91.  With a head's pages after each other
// instead of a page's heads that was 99, and 500 MB read for 261: the table, 10 MB, outgrew the L2s between two heads.
// In fp64 alone: fp32 keys, 633 MB with the table, 149 by neighbouring pairs and 181 half-split (128 as they are, 4.9 TB/s); half-split
// pairs through LDS, 60 of them, 203 in bf16 and 290 in fp32.
template <int DT, int D, int MODE, int THREADS, int N>
__global__ __launch_bounds__(THREADS, MODE == KEY_HALF_ANY || (N == 4 && THREADS == 512) ? 2 : 4) void kv_append_kernel(const AppendArgs a) {
  constexpr int L = D / 8, T = THREADS / L, WAVES = THREADS / 64;  // lanes a token, tokens a step
  constexpr bool QUICK = DT != MXF8_F32 && (MODE == KEY_PAIRS || MODE == KEY_HALF);
  __shared__ uint32_t red[2][WAVES];
  __shared__ float exchange[MODE == KEY_HALF_ANY ? THREADS * 8 : 1];
  const int b = blockIdx.z, lane = threadIdx.x & 63, l = threadIdx.x % L, c0 = 8 * l;
  const int page = 1 << a.c.shift;
  // Every eighth page to one XCD with all its heads, so that its L2 holds the page's cos / sin for them
  uint32_t p = blockIdx.x, h = blockIdx.y;
  if (a.eights) {
    const uint32_t id = blockIdx.y * gridDim.x + blockIdx.x, H = a.c.H, group = id / (8 * H), r = id - group * 8 * H;
    const bool whole = group < (uint32_t)a.eights;
    h = whole ? r / 8 : r % H;
    p = 8 * group + (whole ? r % 8 : r / H);
  }
  const int64_t start = a.starts[b];
  const int64_t count = a.counts ? min(max(a.counts[b], 0), a.S) : a.S;
  const int64_t index = (start >> a.c.shift) + p, base = index << a.c.shift;
  const int64_t lo = max(max(start, base), (int64_t)0), hi = min(start + count, base + page);
  if (lo >= hi || index >= a.c.width) return;
  const int pid = kv_page(a.c, b, (int)index);
  if (pid < 0) return;
  const bool any_old = start > base;
  const int first = threadIdx.x / L;  // this thread's tokens of the page: first, first + T, ...
  bool there[N];
#pragma unroll
  for (int i = 0; i < N; ++i) there[i] = first + i * T < page && base + first + i * T >= lo && base + first + i * T < hi;
  const int64_t s0 = base + first - start;  // of the call's tokens, this thread's first
  const float* turns = a.turns + b * a.turns_batch;
  // half-split: the channel that each of this lane's turns with, and the norm's weights of both
  auto partner = [&](int j) {
    if (MODE == KEY_HALF) return (c0 < a.P ? c0 + a.P : c0 < 2 * a.P ? c0 - a.P : c0) + j;
    const int c = c0 + j;
    return c < a.P ? c + a.P : c < 2 * a.P ? c - a.P : c;
  };
  Raw8<DT> wk, wp;
  wk.fill(1.0f), wp.fill(1.0f);
  if (MODE != KEY_PLAIN && a.w) {
    wk.load(a.w, c0);
    if (MODE == KEY_HALF) wp.load(a.w, partner(0));
  }
  const int plane = (lane - l) + partner(0) / 8;  // the lane that holds all eight
  Raw8<DT> kr[N], vr[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    kr[i].zero(), vr[i].zero();
    if (there[i]) {
      kr[i].load_stream(a.x[0], b * a.xs[0][0] + h * a.xs[0][1] + (s0 + i * T) * a.xs[0][2] + c0);
      vr[i].load_stream(a.x[1], b * a.xs[1][0] + h * a.xs[1][1] + (s0 + i * T) * a.xs[1][2] + c0);
    }
  }
  // interleaved: a lane's four pairs of a token, neighbours in memory
  auto load_turns = [&](int i, float (&cs)[8]) {
    if (MODE != KEY_PAIRS) return;
    // (a token that is not there has zeros, and any angles)
    const float* t = turns + ((there[i] ? s0 + i * T : 0) * a.P + c0 / 2) * 2;
    if (c0 / 2 + 4 <= a.P) {
      const floats4 t0 = *(gfloats4)(gbytes)t, t1 = *(gfloats4)(gbytes)(t + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) cs[j] = t0[j], cs[4 + j] = t1[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) cs[j] = c0 / 2 + j / 2 < a.P ? t[j] : 0.0f;
    }
  };
  float cs[2][8];
  load_turns(0, cs[0]);
  const int64_t ph = (int64_t)pid * a.c.H + h;
  const int old[2] = {(int)a.c.ks[ph] - 127, (int)a.c.vs[ph] - 127};
  // One token's eight channels in fp32, within 13 units of their last place: x w is exact, the turn's second product keeps
  // its rounding error (so that what cancels leaves no more than three half units), and the norm's factor comes last: 14 halves of
  // 2^-23 in its sum, half of that in the root, two for itself, one for the last product.  False where this may
  // decide a code or a scale, within 16 units of a border (see round_keys), or where something over- or underflows.
  auto quick_key = [&](int i, const float (&x)[8], const float (&w)[8], float (&f)[8]) {
    float g = 1.0f, u[8];
    if (a.w) {
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(x[j], x[j], ss);
      g = __builtin_amdgcn_rsqf(__builtin_fmaf(lanes_sum<L>(ss), 1.0f / D, a.eps));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = u[j] = x[j] * w[j];
    // a co + b si
    auto turn = [](float a, float co, float b, float si) {
      const float p = b * si;
      return __builtin_fmaf(a, co, p) + __builtin_fmaf(b, si, -p);
    };
    if constexpr (MODE == KEY_PAIRS) {
#pragma unroll
      for (int j = 0; j < 8; j += 2)
        if (c0 / 2 + j / 2 < a.P) {
          f[j] = turn(u[j], cs[i & 1][j], -u[j + 1], cs[i & 1][j + 1]);
          f[j + 1] = turn(u[j + 1], cs[i & 1][j], u[j], cs[i & 1][j + 1]);
        }
    } else {
      Raw8<DT> r = kr[i];
      r.from_lane(plane);
      float q[8], wq[8];
      r.get(q);
      wp.get(wq);
      if (c0 < 2 * a.P) {
        const float* t = turns + ((there[i] ? s0 + i * T : 0) * a.P + min(c0, partner(0))) * 2;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const floats4 v = *(gfloats4)(gbytes)(t + 2 * j);
          f[j] = turn(u[j], v[0], q[j] * wq[j], c0 < a.P ? -v[1] : v[1]);
          f[j + 1] = turn(u[j + 1], v[2], q[j + 1] * wq[j + 1], c0 < a.P ? -v[3] : v[3]);
        }
      }
    }
    uint32_t near = ~0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[j] *= g;
      near = min(near, (__float_as_uint(f[j]) + 16) << 13);
    }
    // (what is neither normed nor turned is exact)
    return (near > 32u << 13 && g >= 0x1p-40f && g <= 0x1p40f) || (!a.w && c0 >= 2 * a.P);
  };
  float k[N][8];
  uint32_t raw[2] = {0, 0}, top[2];
#pragma unroll
  for (int i = 0; i < N; ++i) raw[0] = raw_max(kr[i], raw[0]), raw[1] = raw_max(vr[i], raw[1]);
  top[0] = raw_max_f32<DT>(raw[0]), top[1] = raw_max_f32<DT>(raw[1]);
  if constexpr (MODE == KEY_PLAIN) {
#pragma unroll
    for (int i = 0; i < N; ++i) kr[i].get(k[i]);
  } else {
    float size = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      __builtin_amdgcn_sched_barrier(0);  // (one token's values at a time)
      if (i + 1 < N) load_turns(i + 1, cs[(i + 1) & 1]);
      if (!__ballot(there[i])) {  // none of this wave's tokens
#pragma unroll
        for (int j = 0; j < 8; ++j) k[i][j] = 0.0f;
        continue;
      }
      float x[8], w[8];
      kr[i].get(x);
      wk.get(w);
      if constexpr (QUICK) {
        const bool sure = quick_key(i, x, w, k[i]);
        if (!__ballot(there[i] && !sure)) {
#pragma unroll
          for (int j = 0; j < 8; ++j) size = fmaxf(size, fabsf(k[i][j]));
          continue;
        }
      }
      // the same in 64 bits, rounded once
      double y[8], g = 1.0;
      if (a.w) {
        double ss = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)x[j], (double)x[j], ss);
        g = rsqrt(__builtin_fma(lanes_sum64<L>(ss), 1.0 / D, (double)a.eps));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = (double)x[j] * (g * (double)w[j]);
      if constexpr (MODE == KEY_PAIRS) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c0 / 2 + j < a.P) {
            const double u = y[2 * j], v = y[2 * j + 1], co = cs[i & 1][2 * j], si = cs[i & 1][2 * j + 1];
            y[2 * j] = __builtin_fma(u, co, -(v * si));
            y[2 * j + 1] = __builtin_fma(u, si, v * co);
          }
      } else {
        float q[8];
        const float* t = turns + (there[i] ? s0 + i * T : 0) * a.P * 2;
        if constexpr (MODE == KEY_HALF) {
          Raw8<DT> r = kr[i];
          r.from_lane(plane);
          r.get(q);
          wp.get(w);
        } else {
          // (this wave's part of the exchange alone: LDS operations of a wave complete in order)
          float* mine = exchange + (threadIdx.x & ~63) * 8;
          *reinterpret_cast<v4f*>(mine + lane * 8) = v4f{x[0], x[1], x[2], x[3]};
          *reinterpret_cast<v4f*>(mine + lane * 8 + 4) = v4f{x[4], x[5], x[6], x[7]};
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int j = 0; j < 8; ++j) q[j] = mine[(lane - l) * 8 + partner(j)];
          __builtin_amdgcn_wave_barrier();
          typedef typename Elem<DT>::T E;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (a.w) w[j] = Elem<DT>::to_f32(static_cast<const E*>(a.w)[partner(j)]);
        }
#pragma unroll
        for (int j4 = 0; j4 < 8; j4 += 2) {
          float co[2], si[2];
          if (MODE == KEY_HALF && c0 < 2 * a.P) {  // this lane's pairs are neighbours
            const floats4 v = *(gfloats4)(gbytes)(t + (min(c0, partner(0)) + j4) * 2);
            co[0] = v[0], si[0] = v[1], co[1] = v[2], si[1] = v[3];
          } else {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              const int pair = min(c0 + j4 + m, partner(j4 + m));
              co[m] = pair < a.P ? t[2 * pair] : 1.0f, si[m] = pair < a.P ? t[2 * pair + 1] : 0.0f;
            }
          }
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const int j = j4 + m;
            if (c0 + j < 2 * a.P)
              y[j] = __builtin_fma(y[j], (double)co[m], (double)q[j] * (g * (double)w[j]) * (double)(c0 + j < a.P ? -si[m] : si[m]));
          }
        }
      }
      round_keys(y, k[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) size = fmaxf(size, fabsf(k[i][j]));
    }
    // (what is not finite before the turn stays so, but a maximum leaves NaN out)
    top[0] = max(__float_as_uint(size), top[0] >= INF_BITS ? top[0] : 0);
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    top[p] = wave_max_u32(top[p]);
    if (lane == 0) red[p][threadIdx.x >> 6] = top[p];
  }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < 2; ++p)
    top[p] = block_max(red[p]);
  uint8_t* code[2] = {const_cast<uint8_t*>(a.c.k) + (ph << a.c.shift) * D, const_cast<uint8_t*>(a.c.v) + (ph << a.c.shift) * D};
  int e[2];
  if (max(top[0], top[1]) <= LARGEST_BITS) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      e[p] = kv_exponent(__uint_as_float(top[p]));
      if (any_old) e[p] = max(e[p], old[p]);
    }
    const float sk = kv_pow2(e[0]), sv = kv_pow2(e[1]);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (there[i]) {
        const int64_t o = (int64_t)(first + i * T) * D + c0;
        *reinterpret_cast<v2i*>(code[0] + o) = codes_of(k[i], sk);
        *reinterpret_cast<v2i*>(code[1] + o) = codes_of<DT>(vr[i], sv);
      }
  } else {
    // Something is not finite, or past the scales' range: the largest finite size, infinities as the largest code.  A NaN
    // anywhere in a token stays as one in its key, which reaches the rows that attend to it and no others; a NaN among
    // the values would reach every row of a product, also those whose mask leaves it out.
    float size[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float v[8];
      vr[i].get(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = fabsf(k[i][j]), y = fabsf(v[j]);
        size[0] = fmaxf(size[0], x < INFINITY ? x : 0.0f), size[1] = fmaxf(size[1], y < INFINITY ? y : 0.0f);
      }
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      top[p] = wave_max_u32(__float_as_uint(size[p]));
      if (lane == 0) red[p][threadIdx.x >> 6] = top[p];
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      e[p] = kv_exponent(__uint_as_float(block_max(red[p])));
      if (any_old) e[p] = max(e[p], old[p]);
    }
    const float ik = kv_pow2(-e[0]), iv = kv_pow2(-e[1]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float v[8];
      vr[i].get(v);
      bool bad = false;
      uint32_t w[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = p < 2 ? k[i][4 * p + j] : v[4 * (p - 2) + j];
          bad |= x[j] != x[j];
          x[j] = x[j] == x[j] ? clamp448(x[j] * (p < 2 ? ik : iv)) : 0.0f;
        }
        w[p] = cvt4_e4m3(x[0], x[1], x[2], x[3]);
      }
      const uint64_t any = __ballot(bad);
      if (l == 0 && (any >> lane & ((1ull << L) - 1))) w[0] |= 0x7fu;
      if (there[i]) {
        const int64_t o = (int64_t)(first + i * T) * D + c0;
        *reinterpret_cast<v2i*>(code[0] + o) = v2i{(int)w[0], (int)w[1]};
        *reinterpret_cast<v2i*>(code[1] + o) = v2i{(int)w[2], (int)w[3]};
      }
    }
  }
  if (threadIdx.x == 0) {
    const_cast<uint8_t*>(a.c.ks)[ph] = (uint8_t)(e[0] + 127);
    const_cast<uint8_t*>(a.c.vs)[ph] = (uint8_t)(e[1] + 127);
  }
  if (any_old)
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int d = old[p] - e[p];
      if (d >= 0) continue;
      const float s = kv_pow2(max(d, -126));
      for (int64_t o = threadIdx.x * 8; o < (start - base) * D; o += THREADS * 8) {
        v2i w = *reinterpret_cast<const v2i*>(code[p] + o);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const v2f x = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], false), y = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], true);
          w[j] = (int)cvt4_e4m3(x[0] * s, x[1] * s, y[0] * s, y[1] * s);
        }
        *reinterpret_cast<v2i*>(code[p] + o) = w;
      }
    }
}

template <int DT, int D, int MODE>
static int launch_append(const AppendArgs& a, dim3 grid, hipStream_t st) {
  // Pages of 1024 chunks: four tokens a lane in workgroups of 256, or, where these are few or the registers do not hold
  // them, two in 512.  us of four / two, 24 heads of 128 in bf16, pages of 64 tokens:
  //   workgroups        120        408         624          792          1056         2088         7632
  //   plain keys        4.8 / 4.5  5.6 / 5.7   7.1 / 7.1    8.3 / 8.2    11.4 / 11.5  21.4 / 22.9  65 / 70
  //   normed, pairs     7.3 / 6.1  8.7 / 8.1   10.4 / 11.4  11.8 / 13.6  15.6 / 16.1  26.8 / 28.5  79 / 82
  //   normed, halves    9.2 / 7.1  10.0 / 9.7  11.5 / 12.9  13.5 / 15.8  17.6 / 19.4  30.2 / 33.8  91 / 102
  // Turned keys take 86 or 102 registers with two tokens a lane, so that 512 workgroups are a round; from there to 1024 four
  // are 9-15% faster, and of 64 channels 4-14% slower at 624.
  const int chunks = (D << a.c.shift) / 8;  // of eight channels
  const int64_t blocks = (int64_t)grid.x * grid.y * grid.z;
  if (chunks <= 256) {
    kv_append_kernel<DT, D, MODE, 256, 1><<<grid, 256, 0, st>>>(a);
  } else if (chunks == 512) {
    kv_append_kernel<DT, D, MODE, 256, 2><<<grid, 256, 0, st>>>(a);
  } else if (chunks == 1024) {
    if constexpr (MODE == KEY_PLAIN || (MODE != KEY_HALF_ANY && DT != MXF8_F32)) {
      if (blocks >= 1024) {
        kv_append_kernel<DT, D, MODE, 256, 4><<<grid, 256, 0, st>>>(a);
        return check_launch("kv_append");
      }
    }
    kv_append_kernel<DT, D, MODE, 512, 2><<<grid, 512, 0, st>>>(a);
  } else if constexpr (D == 128) {
    kv_append_kernel<DT, D, MODE, 512, 4><<<grid, 512, 0, st>>>(a);
  }
  return check_launch("kv_append");
}
template <int DT, int D>
static int launch_append(const AppendArgs& a, int mode, dim3 grid, hipStream_t st) {
  switch (mode) {
    case KEY_PLAIN: return launch_append<DT, D, KEY_PLAIN>(a, grid, st);
    case KEY_PAIRS: return launch_append<DT, D, KEY_PAIRS>(a, grid, st);
    case KEY_HALF: return launch_append<DT, D, KEY_HALF>(a, grid, st);
    default: return launch_append<DT, D, KEY_HALF_ANY>(a, grid, st);
  }
}

struct ReadArgs {
  KvPages c;
  const int32_t *starts, *lengths;
  void *k, *v;
  int64_t T, pages;  // tokens of a sequence, and the pages that they may touch
};

// Eight channels a lane, so that a wave stores a row of memory at once; a page and head is 128 such chunks or a multiple, and
// each wave reads chunks of one page, of keys and of values, I times.  Bound by memory: 20280 tokens x 24 heads x 128, 374 MB,
// 54 us (a part of it from the last cache; 16 channels a lane, two stores of half a row, 133).
template <int DT, int D, int I>
__global__ __launch_bounds__(256) void kv_read_kernel(const ReadArgs a) {
  constexpr int L = D / 8;
  const int b = blockIdx.z, h = blockIdx.y, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int per = a.c.shift + (D == 128 ? 4 : 3) - 6;  // log2 of the waves' turns that a page takes
  const int64_t start = a.starts[b], first = start >> a.c.shift;
  const int64_t end = min(start + a.T, (int64_t)kv_length(a.c, a.lengths ? (int64_t)a.lengths[b] : INT64_MAX));
  v2i x[I][2];
  float s[I][2];
  int64_t at[I];
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int64_t turn = (int64_t)(blockIdx.x * I + i) * 4 + w, index = first + (turn >> per);
    const int slot = ((int)(turn & ((1 << per) - 1)) * 64 + lane) / L;
    const int64_t pos = (index << a.c.shift) + slot;
    at[i] = (turn >> per) < a.pages && pos >= start && pos < start + a.T ? pos - start : -1;
    int pid = -1;
    if ((index << a.c.shift) < end && index >= 0) {
      pid = kv_entry(a.c, b, (int)index);
      pid = kv_valid(a.c, pid) ? pid : -1;
    }
    const int64_t ph = (int64_t)max(pid, 0) * a.c.H + h;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      x[i][p] = v2i{0, 0}, s[i][p] = 0.0f;
      if (pid >= 0) {
        s[i][p] = kv_scale((p ? a.c.vs : a.c.ks)[ph]);
        if (at[i] >= 0 && pos < end)
          x[i][p] = *reinterpret_cast<const v2i*>((p ? a.c.v : a.c.k) + ((ph << a.c.shift) + slot) * D + lane % L * 8);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < I; ++i) {
    if (at[i] < 0) continue;
    const int64_t o = (((int64_t)b * a.c.H + h) * a.T + at[i]) * D + lane % L * 8;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const v2f u = __builtin_amdgcn_cvt_pk_f32_fp8(x[i][p][j], false), v = __builtin_amdgcn_cvt_pk_f32_fp8(x[i][p][j], true);
        f[4 * j] = u[0] * s[i][p], f[4 * j + 1] = u[1] * s[i][p], f[4 * j + 2] = v[0] * s[i][p], f[4 * j + 3] = v[1] * s[i][p];
      }
      Raw8<DT> r;
      r.set(f);
      r.stream(p ? a.v : a.k, o);
    }
  }
}

}  // namespace mxf8

using namespace mxf8;

extern "C" int mxf8_kv_append(const void* k, const int64_t k_strides[4], const void* v, const int64_t v_strides[4],
                              int dtype, int64_t B, int64_t H, int64_t S, int64_t D, const float* turns,
                              int64_t turns_batch_stride, int64_t P, const void* k_weight, float eps, int interleaved,
                              const int32_t* page_table, int64_t table_stride, int64_t table_width,
                              const int32_t* starts, const int32_t* counts, uint8_t* k_codes, uint8_t* v_codes,
                              uint8_t* k_scale, uint8_t* v_scale, int64_t pages, int64_t page_size,
                              hipStream_t stream) {
  const char* what = "kv_append";
  AppendArgs a{};
  if (const int rc = kv_check_pages(what, k_codes, v_codes, k_scale, v_scale, pages, H, page_size, D, page_table,
                                    table_stride, table_width, B, &a.c))
    return rc;
  if (S < 0 || S > (1 << 30)) return set_error(MXF8_EINVAL, "%s: bad shape", what);
  if (P < 0 || 2 * P > D)
    return set_error(MXF8_EINVAL, "%s: %lld pairs do not fit D=%lld", what, (long long)P, (long long)D);
  if (dtype != MXF8_BF16 && dtype != MXF8_F16 && dtype != MXF8_F32)
    return set_error(MXF8_EINVAL, "%s: bad dtype %d", what, dtype);
  if (!(eps >= 0.0f)) return set_error(MXF8_EINVAL, "%s: eps must be >= 0", what);
  if (B == 0 || H == 0 || S == 0 || table_width == 0 || pages == 0) return MXF8_OK;
  if (!k || !v || !k_strides || !v_strides || !starts || (P && !turns))
    return set_error(MXF8_EINVAL, "%s: null pointer", what);
  if ((uintptr_t)turns % 8 || turns_batch_stride % 2)
    return set_error(MXF8_EINVAL, "%s: table must be 8-byte aligned", what);
  if (k_strides[3] != 1 || v_strides[3] != 1) return set_error(MXF8_EINVAL, "%s: channels must be contiguous", what);
  a.x[0] = k, a.x[1] = v, a.w = k_weight;
  for (int i = 0; i < 3; ++i) a.xs[0][i] = k_strides[i], a.xs[1][i] = v_strides[i];
  a.turns = turns, a.turns_batch = turns_batch_stride;
  a.starts = starts, a.counts = counts;
  a.S = (int)S, a.P = (int)P, a.eps = eps;
  const int mode = P == 0 && !k_weight ? KEY_PLAIN : P == 0 || interleaved ? KEY_PAIRS : P % 8 == 0 ? KEY_HALF : KEY_HALF_ANY;
  // a run of S tokens touches up to so many pages, wherever it starts
  const int64_t touched = (S + page_size - 2) / page_size + 1;
  if (!grid_fits(touched, 512)) return set_error(MXF8_EINVAL, "%s: shape too large", what);
  a.eights = touched * H < (1 << 30) ? (int)(touched / 8) : 0;
  const dim3 grid((unsigned)touched, (unsigned)H, (unsigned)B);
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return D == 128 ? launch_append<DT, 128>(a, mode, grid, stream) : launch_append<DT, 64>(a, mode, grid, stream);
  };
  return dtype == MXF8_BF16  ? launch(std::integral_constant<int, MXF8_BF16>{})
         : dtype == MXF8_F16 ? launch(std::integral_constant<int, MXF8_F16>{})
                             : launch(std::integral_constant<int, MXF8_F32>{});
}

extern "C" int mxf8_kv_read(const uint8_t* k_codes, const uint8_t* v_codes, const uint8_t* k_scale,
                            const uint8_t* v_scale, int64_t pages, int64_t H, int64_t page_size, int64_t D,
                            const int32_t* page_table, int64_t table_stride, int64_t table_width, int64_t B,
                            const int32_t* starts, int64_t T, const int32_t* lengths, void* k, void* v, int dtype,
                            hipStream_t stream) {
  const char* what = "kv_read";
  ReadArgs a{};
  if (const int rc = kv_check_pages(what, k_codes, v_codes, k_scale, v_scale, pages, H, page_size, D, page_table,
                                    table_stride, table_width, B, &a.c))
    return rc;
  if (T < 0 || T > (1 << 30)) return set_error(MXF8_EINVAL, "%s: bad shape", what);
  if (dtype != MXF8_BF16 && dtype != MXF8_F16 && dtype != MXF8_F32)
    return set_error(MXF8_EINVAL, "%s: bad dtype %d", what, dtype);
  if (B == 0 || H == 0 || T == 0) return MXF8_OK;
  if (!starts || !k || !v) return set_error(MXF8_EINVAL, "%s: null pointer", what);
  a.starts = starts, a.lengths = lengths, a.k = k, a.v = v;
  a.T = T, a.pages = (T + page_size - 2) / page_size + 1;
  // four turns of a wave in flight together where there are enough to go round
  const int64_t turns = a.pages * (page_size * D / 512);
  const bool many = turns * H * B >= 4 * 4096;
  const int64_t blocks = cdiv(turns, many ? 16 : 4);
  if (!grid_fits(blocks, 256)) return set_error(MXF8_EINVAL, "%s: shape too large", what);
  const dim3 grid((unsigned)blocks, (unsigned)H, (unsigned)B);
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (D == 128)
      many ? kv_read_kernel<DT, 128, 4><<<grid, 256, 0, stream>>>(a) : kv_read_kernel<DT, 128, 1><<<grid, 256, 0, stream>>>(a);
    else
      many ? kv_read_kernel<DT, 64, 4><<<grid, 256, 0, stream>>>(a) : kv_read_kernel<DT, 64, 1><<<grid, 256, 0, stream>>>(a);
    return check_launch(what);
  };
  return dtype == MXF8_BF16  ? launch(std::integral_constant<int, MXF8_BF16>{})
         : dtype == MXF8_F16 ? launch(std::integral_constant<int, MXF8_F16>{})
                             : launch(std::integral_constant<int, MXF8_F32>{});
}
