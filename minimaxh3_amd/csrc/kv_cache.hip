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

enum { TURN_NONE, TURN_INTERLEAVED, TURN_HALF, TURN_HALF_ANY };

struct AppendArgs {
  KvPages c;
  const void *x[2], *w;   // keys and values; the key norm's weight or null
  int64_t xs[2][3];       // strides of batch, head, token
  const float* turns;     // cos / sin [.., S, P, 2]
  int64_t turns_batch;
  const int32_t *starts, *counts;
  int S, P, mode, heads;  // heads: of one workgroup
  float eps;
};

// A workgroup writes one page of one sequence, head after head: D / 8 lanes hold a token's eight channels each, so the
// page's maximum is one reduction over values that stay in registers until they are rounded.
template <int DT, int D, int N>
__global__ __launch_bounds__(256) void kv_append_kernel(const AppendArgs a) {
  constexpr int L = D / 8, T = 256 / L;  // lanes a token, tokens a step
  __shared__ float red[2][2][4];
  __shared__ float exchange[256 * 8];
  const int b = blockIdx.z, lane = threadIdx.x & 63, l = threadIdx.x % L, c0 = 8 * l;
  const int page = 1 << a.c.shift;
  const int64_t start = a.starts[b];
  const int64_t count = a.counts ? min(max(a.counts[b], 0), a.S) : a.S;
  const int64_t index = (start >> a.c.shift) + blockIdx.x, base = index << a.c.shift;
  const int64_t lo = max(max(start, base), (int64_t)0), hi = min(start + count, base + page);
  if (lo >= hi || index >= a.c.width) return;
  const int pid = kv_page(a.c, b, (int)index);
  if (pid < 0) return;
  const bool any_old = start > base;
  const int first = threadIdx.x / L;  // this thread's tokens of the page: first, first + T, ...
  const float* turns = a.turns + b * a.turns_batch;
  float wk[8], wp[8];
  // half-split partner: channel c +- P, in lane l +- P / 8 of the token where P % 8 == 0
  const int plane = (lane - l) + min(max(c0 < a.P ? l + a.P / 8 : l - a.P / 8, 0), L - 1);
  if (a.w) {
    Raw8<DT> w;
    w.load(a.w, c0);
    w.get(wk);
    if (a.mode == TURN_HALF) w.from_lane(plane);
    w.get(wp);
  }
  for (int h = blockIdx.y * a.heads, last = min(h + a.heads, a.c.H), turn = 0; h < last; ++h, turn ^= 1) {
    Raw8<DT> kr[N], vr[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t pos = base + first + i * T;
      kr[i].zero(), vr[i].zero();
      if (first + i * T < page && pos >= lo && pos < hi) {
        const int64_t s = pos - start;
        kr[i].load_stream(a.x[0], b * a.xs[0][0] + h * a.xs[0][1] + s * a.xs[0][2] + c0);
        vr[i].load_stream(a.x[1], b * a.xs[1][0] + h * a.xs[1][1] + s * a.xs[1][2] + c0);
      }
    }
    const int64_t ph = (int64_t)pid * a.c.H + h;
    const int ek_old = (int)a.c.ks[ph] - 127, ev_old = (int)a.c.vs[ph] - 127;
    float k[N][8], amax[2] = {0.0f, 0.0f};
    bool bad[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t pos = base + first + i * T;
      const bool there = first + i * T < page && pos >= lo && pos < hi;
      float f[8], q[8];
      kr[i].get(f);
      if (a.mode == TURN_HALF) kr[i].from_lane(plane);
      kr[i].get(q);
      if (a.w) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(f[j], f[j], ss);
        const float r = rsqrtf(__builtin_fmaf(lanes_sum<L>(ss), 1.0f / D, a.eps));
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= r * wk[j], q[j] *= r * wp[j];
      }
      const float2* t = reinterpret_cast<const float2*>(turns) + (there ? pos - start : 0) * a.P;
      if (a.mode == TURN_INTERLEAVED) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = f[2 * j], y = f[2 * j + 1];
          if (c0 / 2 + j < a.P) {
            const float2 cs = t[c0 / 2 + j];
            f[2 * j] = __builtin_fmaf(x, cs.x, -(y * cs.y));
            f[2 * j + 1] = __builtin_fmaf(x, cs.y, y * cs.x);
          }
        }
      } else if (a.mode != TURN_NONE) {
        if (a.mode == TURN_HALF_ANY) {
          // (this wave's part of the exchange alone: LDS operations of a wave complete in order)
          float* mine = exchange + (threadIdx.x & ~63) * 8;
          *reinterpret_cast<v4f*>(mine + lane * 8) = v4f{f[0], f[1], f[2], f[3]};
          *reinterpret_cast<v4f*>(mine + lane * 8 + 4) = v4f{f[4], f[5], f[6], f[7]};
          __builtin_amdgcn_wave_barrier();
          const float* head = mine + (lane - l) * 8;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int c = c0 + j;
            q[j] = head[c < a.P ? c + a.P : c < 2 * a.P ? c - a.P : c];
          }
          __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = c0 + j;
          if (c < 2 * a.P) {
            const float2 cs = t[c < a.P ? c : c - a.P];
            f[j] = __builtin_fmaf(f[j], cs.x, q[j] * (c < a.P ? -cs.y : cs.y));
          }
        }
      }
      bad[i] = false;
      float v[8];
      vr[i].get(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        k[i][j] = f[j];
        const float x = fabsf(f[j]), y = fabsf(v[j]);
        amax[0] = fmaxf(amax[0], x < INFINITY ? x : 0.0f);
        amax[1] = fmaxf(amax[1], y < INFINITY ? y : 0.0f);
        bad[i] |= !(x <= INFINITY) || !(y <= INFINITY);
      }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      amax[p] = lanes_max<64>(amax[p]);
      if (lane == 0) red[turn][p][threadIdx.x >> 6] = amax[p];
    }
    __syncthreads();  // (the two halves of `red` in turn: the next head's writes pass this one's reads by a barrier)
    int e[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      e[p] = kv_exponent(fmaxf(fmaxf(red[turn][p][0], red[turn][p][1]), fmaxf(red[turn][p][2], red[turn][p][3])));
      if (any_old) e[p] = max(e[p], p ? ev_old : ek_old);
    }
    const float ik = kv_pow2(-e[0]), iv = kv_pow2(-e[1]);
    uint8_t* kc = const_cast<uint8_t*>(a.c.k) + (ph << a.c.shift) * D;
    uint8_t* vc = const_cast<uint8_t*>(a.c.v) + (ph << a.c.shift) * D;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t pos = base + first + i * T;
      float v[8];
      vr[i].get(v);
      // A NaN anywhere in the token stays as one in its key, which reaches the rows that attend to it and no others;
      // a NaN among the values would reach every row of a product, also those whose mask leaves it out.
      const uint64_t any_bad = __ballot(bad[i]);
      uint32_t nan_key = 0;
      if (any_bad) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          k[i][j] = k[i][j] == k[i][j] ? k[i][j] : 0.0f;
          v[j] = v[j] == v[j] ? v[j] : 0.0f;
        }
        nan_key = l == 0 && (any_bad >> (lane - l) & ((1ull << L) - 1)) ? 0x7fu : 0u;
      }
      if (first + i * T < page && pos >= lo && pos < hi) {
        uint32_t w[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const float* x = p < 2 ? k[i] + 4 * p : v + 4 * (p - 2);
          const float s = p < 2 ? ik : iv;
          w[p] = cvt4_e4m3(clamp448(x[0] * s), clamp448(x[1] * s), clamp448(x[2] * s), clamp448(x[3] * s));
        }
        w[0] |= nan_key;
        const int64_t o = (int64_t)(first + i * T) * D + c0;
        *reinterpret_cast<v2i*>(kc + o) = v2i{(int)w[0], (int)w[1]};
        *reinterpret_cast<v2i*>(vc + o) = v2i{(int)w[2], (int)w[3]};
      }
    }
    if (threadIdx.x == 0) {
      const_cast<uint8_t*>(a.c.ks)[ph] = (uint8_t)(e[0] + 127);
      const_cast<uint8_t*>(a.c.vs)[ph] = (uint8_t)(e[1] + 127);
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int d = (p ? ev_old : ek_old) - e[p];
      if (!any_old || d >= 0) continue;
      const float s = kv_pow2(max(d, -126));
      uint8_t* c = p ? vc : kc;
      for (int64_t o = threadIdx.x * 8; o < (start - base) * D; o += 256 * 8) {
        v2i w = *reinterpret_cast<const v2i*>(c + o);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const v2f x = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], false), y = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], true);
          w[j] = (int)cvt4_e4m3(x[0] * s, x[1] * s, y[0] * s, y[1] * s);
        }
        *reinterpret_cast<v2i*>(c + o) = w;
      }
    }
  }
}

template <int DT, int D>
static int launch_append(AppendArgs& a, dim3 grid, hipStream_t st) {
  const int steps = (D << a.c.shift) / 2048;
  if (steps <= 1)
    kv_append_kernel<DT, D, 1><<<grid, 256, 0, st>>>(a);
  else if (steps == 2)
    kv_append_kernel<DT, D, 2><<<grid, 256, 0, st>>>(a);
  else if (steps == 4)
    kv_append_kernel<DT, D, 4><<<grid, 256, 0, st>>>(a);
  else if constexpr (D == 128)
    kv_append_kernel<DT, D, 8><<<grid, 256, 0, st>>>(a);
  return check_launch("kv_append");
}

struct ReadArgs {
  KvPages c;
  const int32_t *starts, *lengths;
  void *k, *v;
  int64_t T, chunks;  // tokens of a sequence, and its chunks of 16 channels
};

// 16 channels of a token, of keys and of values, per thread.
template <int DT, int D>
__global__ __launch_bounds__(256) void kv_read_kernel(const ReadArgs a) {
  constexpr int L = D / 16;
  const int b = blockIdx.z, h = blockIdx.y;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.chunks) return;
  const int64_t t = i / L, c = i % L * 16, pos = a.starts[b] + t;
  int pid = -1;
  if (pos >= 0 && pos < kv_length(a.c, a.lengths ? (int64_t)a.lengths[b] : INT64_MAX))
    pid = kv_page(a.c, b, (int)(pos >> a.c.shift));
  const int64_t ph = (int64_t)max(pid, 0) * a.c.H + h, o = ((int64_t)b * a.c.H + h) * a.T * D + t * D + c;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    v4i w = {0, 0, 0, 0};
    float s = 0.0f;
    if (pid >= 0) {
      w = *reinterpret_cast<const v4i*>((p ? a.c.v : a.c.k) + ((ph << a.c.shift) + (pos & ((1 << a.c.shift) - 1))) * D + c);
      s = kv_scale((p ? a.c.vs : a.c.ks)[ph]);
    }
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const v2f x = __builtin_amdgcn_cvt_pk_f32_fp8(w[2 * g + j], false);
        const v2f y = __builtin_amdgcn_cvt_pk_f32_fp8(w[2 * g + j], true);
        f[4 * j] = x[0] * s, f[4 * j + 1] = x[1] * s, f[4 * j + 2] = y[0] * s, f[4 * j + 3] = y[1] * s;
      }
      Raw8<DT> r;
      r.set(f);
      r.stream(p ? a.v : a.k, o + 8 * g);
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
  a.mode = P == 0 ? TURN_NONE : interleaved ? TURN_INTERLEAVED : P % 8 == 0 ? TURN_HALF : TURN_HALF_ANY;
  a.heads = 1;
  // a run of S tokens touches up to so many pages, wherever it starts
  const int64_t touched = (S + page_size - 2) / page_size + 1;
  if (!grid_fits(touched, 256)) return set_error(MXF8_EINVAL, "%s: shape too large", what);
  const dim3 grid((unsigned)touched, (unsigned)cdiv(H, a.heads), (unsigned)B);
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return D == 128 ? launch_append<DT, 128>(a, grid, stream) : launch_append<DT, 64>(a, grid, stream);
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
  a.T = T, a.chunks = T * (D / 16);
  if (!grid_fits(cdiv(a.chunks, 256), 256)) return set_error(MXF8_EINVAL, "%s: shape too large", what);
  const dim3 grid((unsigned)cdiv(a.chunks, 256), (unsigned)H, (unsigned)B);
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (D == 128)
      kv_read_kernel<DT, 128><<<grid, 256, 0, stream>>>(a);
    else
      kv_read_kernel<DT, 64><<<grid, 256, 0, stream>>>(a);
    return check_launch(what);
  };
  return dtype == MXF8_BF16  ? launch(std::integral_constant<int, MXF8_BF16>{})
         : dtype == MXF8_F16 ? launch(std::integral_constant<int, MXF8_F16>{})
                             : launch(std::integral_constant<int, MXF8_F32>{});
}
