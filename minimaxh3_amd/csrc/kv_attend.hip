// Attention over a paged e4m3 cache of keys and values.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij, p_ij = exp(scale q_i . k_j), over the keys j that row i sees
#include <type_traits>

#include "kv_cache.h"
#include "rowio.h"

namespace mxf8 {

struct AttendArgs {
  KvPages c;
  const void* q;
  void* o;
  int64_t qs[3], os[3];  // strides of batch, head, token
  const int32_t *lengths, *q_lengths;
  int B, H, S, causal;
  float scale;  // times log2 e
};

// One wave a row.
template <int DT, int D>
__global__ __launch_bounds__(256) void kv_attend_row_kernel(const AttendArgs a) {
  __shared__ float qrow[4][D];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * 4 + w;
  const int h = blockIdx.y, b = blockIdx.z;
  if (row >= a.S) return;
  const int len = kv_length(a.c, a.lengths[b]);
  const int qlen = a.q_lengths ? min(max(a.q_lengths[b], 0), a.S) : a.S;
  const int64_t seen = row >= qlen ? 0 : a.causal ? (int64_t)len - qlen + row + 1 : len;
  const int hk = h / (a.H / a.c.H);
  typedef typename Elem<DT>::T T;
  const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + h * a.qs[1] + row * a.qs[2];
  for (int d = lane; d < D; d += 64) qrow[w][d] = Elem<DT>::to_f32(q[d]);
  __builtin_amdgcn_wave_barrier();
  float m = -1e30f, l = 0.0f, o[D / 64] = {};
  for (int64_t key0 = 0; key0 < seen; key0 += 64) {
    const int64_t key = key0 + lane;
    const int pid = key < seen ? kv_page(a.c, b, (int)(key >> a.c.shift)) : -1;
    const int64_t ph = (int64_t)max(pid, 0) * a.c.H + hk;
    const int64_t at = ((ph << a.c.shift) + (key & ((1 << a.c.shift) - 1))) * D;
    float x = -1e30f, vs = 0.0f;
    if (pid >= 0) {
      x = 0.0f;
      const int* k = reinterpret_cast<const int*>(a.c.k + at);
      for (int d = 0; d < D; d += 4) {
        const v2f u = __builtin_amdgcn_cvt_pk_f32_fp8(k[d / 4], false), v = __builtin_amdgcn_cvt_pk_f32_fp8(k[d / 4], true);
        x += u[0] * qrow[w][d] + u[1] * qrow[w][d + 1] + v[0] * qrow[w][d + 2] + v[1] * qrow[w][d + 3];
      }
      x *= kv_scale(a.c.ks[ph]) * a.scale;
      vs = kv_scale(a.c.vs[ph]);
    }
    const float mn = fmaxf(m, wave_max(x)), alpha = __builtin_amdgcn_exp2f(m - mn);
    const float p = pid >= 0 ? __builtin_amdgcn_exp2f(x - mn) : 0.0f;
    m = mn;
    l = l * alpha + p;
    for (int i = 0; i < D / 64; ++i) o[i] *= alpha;
    const uint32_t offset_lo = (uint32_t)at, offset_hi = (uint32_t)(at >> 32);
    for (int j = 0; j < 64; ++j) {
      const float pj = __shfl(p * vs, j, 64);
      const int64_t atj = (int64_t)((uint64_t)(uint32_t)__shfl(offset_hi, j, 64) << 32 | (uint32_t)__shfl(offset_lo, j, 64));
      if (__shfl(pid, j, 64) < 0) continue;
      for (int i = 0; i < D / 64; ++i)
        o[i] += pj * __builtin_amdgcn_cvt_f32_fp8(a.c.v[atj + lane + 64 * i], 0);
    }
  }
  l = wave_sum(l);
  const float r = l == 0.0f ? 0.0f : 1.0f / l;
  T* out = static_cast<T*>(a.o) + b * a.os[0] + h * a.os[1] + row * a.os[2];
  for (int i = 0; i < D / 64; ++i) out[lane + 64 * i] = (T)cvt_pk_16<DT>(o[i] * r, 0.0f);
}

}  // namespace mxf8

using namespace mxf8;

extern "C" int64_t mxf8_kv_attend_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t S, int64_t D,
                                                  int64_t table_width, int64_t page_size) {
  return 0;
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
  if (H < 0 || H > 65535 || S < 0 || S > (1 << 30)) return set_error(MXF8_EINVAL, "%s: bad shape", what);
  if (H && (Hk == 0 || H % Hk))
    return set_error(MXF8_EINVAL, "%s: %lld heads over %lld key heads", what, (long long)H, (long long)Hk);
  if (dtype != MXF8_BF16 && dtype != MXF8_F16) return set_error(MXF8_EINVAL, "%s: bad dtype %d", what, dtype);
  if (!__builtin_isfinite(scale)) return set_error(MXF8_EINVAL, "%s: scale must be finite", what);
  if (B == 0 || H == 0 || S == 0) return MXF8_OK;
  if (!q || !out || !q_strides || !out_strides || !lengths) return set_error(MXF8_EINVAL, "%s: null pointer", what);
  if (q_strides[3] != 1 || out_strides[3] != 1)
    return set_error(MXF8_EINVAL, "%s: channels must be contiguous", what);
  a.q = q, a.o = out;
  for (int i = 0; i < 3; ++i) a.qs[i] = q_strides[i], a.os[i] = out_strides[i];
  a.lengths = lengths, a.q_lengths = q_lengths;
  a.B = (int)B, a.H = (int)H, a.S = (int)S, a.causal = causal != 0;
  a.scale = scale * 1.4426950408889634f;
  if (!grid_fits(cdiv(S, 4), 256)) return set_error(MXF8_EINVAL, "%s: shape too large", what);
  const dim3 grid((unsigned)cdiv(S, 4), (unsigned)H, (unsigned)B);
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (D == 128)
      kv_attend_row_kernel<DT, 128><<<grid, 256, 0, stream>>>(a);
    else
      kv_attend_row_kernel<DT, 64><<<grid, 256, 0, stream>>>(a);
    return check_launch(what);
  };
  return dtype == MXF8_BF16 ? launch(std::integral_constant<int, MXF8_BF16>{})
                            : launch(std::integral_constant<int, MXF8_F16>{});
}
