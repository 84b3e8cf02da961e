// Quantization to and from blocks of 32 four-bit values (mxfp4.h).
#include "mxfp4.h"
#include "rowio.h"

namespace mxf8 {

// Both kernels move what they must and little else: 2 bytes in and 0.53 out per element, or the reverse.
// A lane holds 8 elements (a 16-byte load, 4 bytes of codes), a quad of lanes one block, a wave 512 elements.
constexpr int MXQ_ROWS = 4;  // rows per wave: their loads are in flight together

template <int DT>
__global__ __launch_bounds__(256) void mxfp4_quant_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t ldx,
                                                          int64_t M, int K, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales) {
  const int lane = threadIdx.x & 63;
  const int64_t row0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * MXQ_ROWS;
  const int k = (blockIdx.y * 64 + lane) * 8;
  const bool valid = k < K;  // K % 32 == 0: a whole block or none
  const bool pad = !valid && k < (int)mx_slabs(K) * MX_BLOCK * MX_SLAB;
  Raw8<DT> v[MXQ_ROWS];
#pragma unroll
  for (int i = 0; i < MXQ_ROWS; ++i) {
    if (valid && row0 + i < M)
      v[i].load(x, (row0 + i) * ldx + k);
    else
      v[i].zero();
  }
#pragma unroll
  for (int i = 0; i < MXQ_ROWS; ++i) {
    const int64_t m = row0 + i;
    float f[8];
    v[i].get(f);
    const uint32_t byte = mx_scale_byte(mx_block_absmax(f));
    if (m >= M) continue;
    if (valid) *reinterpret_cast<uint32_t*>(codes + m * (K / 2) + k / 2) = mx_codes8(f, byte);
    if ((valid || pad) && (lane & 3) == 0) scales[mx_scale_at(k / MX_BLOCK, m, M)] = (uint8_t)(valid ? byte : 127u);
  }
}

template <int DT>
__global__ __launch_bounds__(256) void mxfp4_dequant_kernel(const uint8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales, int64_t M, int K,
                                                            typename Elem<DT>::T* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int64_t row0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * MXQ_ROWS;
  const int k = (blockIdx.y * 64 + lane) * 8;
  if (k >= K) return;
  uint32_t w[MXQ_ROWS], sb[MXQ_ROWS];
#pragma unroll
  for (int i = 0; i < MXQ_ROWS; ++i) {
    const int64_t m = min(row0 + i, M - 1);
    w[i] = *reinterpret_cast<const uint32_t*>(codes + m * (K / 2) + k / 2);
    sb[i] = scales[mx_scale_at(k / MX_BLOCK, m, M)];
  }
#pragma unroll
  for (int i = 0; i < MXQ_ROWS; ++i) {
    if (row0 + i >= M) break;
    const float s = mx_scale_value(sb[i]);
    const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 0);
    const v2f b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 1);
    const v2f c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 2);
    const v2f d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 3);
    const float f[8] = {a[0] * s, a[1] * s, b[0] * s, b[1] * s, c[0] * s, c[1] * s, d[0] * s, d[1] * s};
    Raw8<DT> o;
    o.set(f);
    o.store(out, (row0 + i) * K + k);
  }
}

static int mx_check(const char* what, int64_t M, int64_t K) {
  if (M < 0 || K <= 0) return set_error(MXF8_EINVAL, "%s: bad shape", what);
  if (K % MX_BLOCK) return set_error(MXF8_EINVAL, "%s: K=%lld must be a multiple of 32", what, (long long)K);
  if (M > 0x7fffffff / 2 || K > (1 << 22)) return set_error(MXF8_EINVAL, "%s: shape too large", what);
  return MXF8_OK;
}

}  // namespace mxf8

using namespace mxf8;

extern "C" int64_t mxf8_mxfp4_scale_bytes(int64_t M, int64_t K) {
  return M <= 0 || K <= 0 ? 0 : mx_slabs(K) * M * MX_SLAB;
}

extern "C" int mxf8_mxfp4_quant(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, uint8_t* codes,
                                uint8_t* scales, hipStream_t stream) {
  if (const int rc = mx_check("mxfp4_quant", M, K)) return rc;
  if (ldx < K && M > 1) return set_error(MXF8_EINVAL, "mxfp4_quant: ldx < K");
  if (M == 0) return MXF8_OK;
  if (!x || !codes || !scales) return set_error(MXF8_EINVAL, "mxfp4_quant: null pointer");
  if ((uintptr_t)codes % 4) return set_error(MXF8_EINVAL, "mxfp4_quant: codes must be 4-byte aligned");
  const dim3 grid((unsigned)cdiv(M, 4 * MXQ_ROWS), (unsigned)cdiv(mx_slabs(K), 2));
  switch (dtype) {
#define MXF8_CASE(DT)                                                                                             \
  case DT:                                                                                                        \
    mxfp4_quant_kernel<DT><<<grid, 256, 0, stream>>>(static_cast<const Elem<DT>::T*>(x), ldx, M, (int)K, codes, scales); \
    break;
    MXF8_CASE(MXF8_BF16)
    MXF8_CASE(MXF8_F16)
    MXF8_CASE(MXF8_F32)
#undef MXF8_CASE
    default: return set_error(MXF8_EINVAL, "mxfp4_quant: bad dtype %d", dtype);
  }
  return check_launch("mxfp4_quant");
}

extern "C" int mxf8_mxfp4_dequant(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, void* out,
                                  int dtype, hipStream_t stream) {
  if (const int rc = mx_check("mxfp4_dequant", M, K)) return rc;
  if (M == 0) return MXF8_OK;
  if (!out || !codes || !scales) return set_error(MXF8_EINVAL, "mxfp4_dequant: null pointer");
  if ((uintptr_t)codes % 4) return set_error(MXF8_EINVAL, "mxfp4_dequant: codes must be 4-byte aligned");
  const dim3 grid((unsigned)cdiv(M, 4 * MXQ_ROWS), (unsigned)cdiv(K, 512));
  switch (dtype) {
#define MXF8_CASE(DT)                                                                                             \
  case DT:                                                                                                        \
    mxfp4_dequant_kernel<DT><<<grid, 256, 0, stream>>>(codes, scales, M, (int)K, static_cast<Elem<DT>::T*>(out)); \
    break;
    MXF8_CASE(MXF8_BF16)
    MXF8_CASE(MXF8_F16)
    MXF8_CASE(MXF8_F32)
#undef MXF8_CASE
    default: return set_error(MXF8_EINVAL, "mxfp4_dequant: bad dtype %d", dtype);
  }
  return check_launch("mxfp4_dequant");
}
