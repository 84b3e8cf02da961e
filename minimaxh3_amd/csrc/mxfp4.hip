// Quantization to and from blocks of 32 four-bit values (mxfp4.h).
#include "mxfp4.h"
#include "rowio.h"

namespace mxf8 {

// Both kernels move what they must and little else: 2 bytes in and 0.53 out per element, or the reverse.
// A lane holds 8 elements (a 16-byte load, 4 bytes of codes), a quad of lanes one block, a wave 512 elements of
// ROWS rows, whose loads are in flight together.  Workgroups go along the rows first, so that those running at the
// same time read and write neighbouring memory (20280 x 12288 bf16: 133 -> 107 us), and past the caches (quantize
// 20280 x 3072 30.4 -> 27.2 us, 5.8 TB/s; back 33.7 -> 25.1, 6.3 TB/s).  A wave spans 512 columns, so a matrix of few leaves
// lanes idle: 62 million elements in rows of 32 take 212 us (back 129), of 288 32 (25), of 1056 32 (28).
constexpr int64_t MX_SMALL = 1 << 24;  // elements up to which two rows and plain loads do (2048 x 3072: 5.5 -> 5.2 us)

// This wave's first row and lane's first column, of workgroups that hold 512 columns of 4 ROWS rows each.
template <int ROWS>
__device__ __forceinline__ int64_t mx_place(int K, int& k) {
  const uint32_t cols = (uint32_t)(K + 511) / 512, rows = blockIdx.x / cols;
  k = ((int)(blockIdx.x - rows * cols) * 64 + (threadIdx.x & 63)) * 8;
  return ((int64_t)rows * 4 + (threadIdx.x >> 6)) * ROWS;
}

template <int DT, int ROWS>
__global__ __launch_bounds__(256) void mxfp4_quant_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t ldx,
                                                          int64_t M, int K, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales) {
  const int lane = threadIdx.x & 63;
  int k;
  const int64_t row0 = mx_place<ROWS>(K, k);
  const bool valid = k < K;  // K % 32 == 0: a whole block or none
  const bool pad = !valid && k < (int)mx_slabs(K) * MX_BLOCK * MX_SLAB;
  Raw8<DT> v[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (!valid || row0 + i >= M)
      v[i].zero();
    else if constexpr (ROWS > 2)
      v[i].load_stream(x, (row0 + i) * ldx + k);
    else
      v[i].load(x, (row0 + i) * ldx + k);
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t m = row0 + i;
    float f[8];
    v[i].get(f);
    const uint32_t byte = mx_scale_byte(mx_block_absmax(f));
    if (m >= M) continue;
    if (valid) *reinterpret_cast<uint32_t*>(codes + m * (K / 2) + k / 2) = mx_codes8(f, byte);
    if ((valid || pad) && (lane & 3) == 0) scales[mx_scale_at(k / MX_BLOCK, m, M)] = (uint8_t)(valid ? byte : 127u);
  }
}

template <int DT, int ROWS>
__global__ __launch_bounds__(256) void mxfp4_dequant_kernel(const uint8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales, int64_t M, int K,
                                                            typename Elem<DT>::T* __restrict__ out) {
  int k;
  const int64_t row0 = mx_place<ROWS>(K, k);
  if (k >= K) return;
  uint32_t w[ROWS], sb[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t m = min(row0 + i, M - 1);
    w[i] = *reinterpret_cast<const uint32_t*>(codes + m * (K / 2) + k / 2);
    sb[i] = scales[mx_scale_at(k / MX_BLOCK, m, M)];
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (row0 + i >= M) break;
    const float s = mx_scale_value(sb[i]);
    const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 0);
    const v2f b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 1);
    const v2f c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 2);
    const v2f d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 3);
    const float f[8] = {a[0] * s, a[1] * s, b[0] * s, b[1] * s, c[0] * s, c[1] * s, d[0] * s, d[1] * s};
    Raw8<DT> o;
    o.set(f);
    o.stream(out, (row0 + i) * K + k);
  }
}

// Workgroups of both: two rows a wave for small matrices, else four.
static bool mx_small(int64_t M, int64_t K) { return M * K <= MX_SMALL; }
static int64_t mx_blocks(int64_t M, int64_t K) { return cdiv(M, mx_small(M, K) ? 8 : 16) * cdiv(K, 512); }

static int mx_check(const char* what, int64_t M, int64_t K) {
  if (M < 0 || K <= 0) return set_error(MXF8_EINVAL, "%s: bad shape", what);
  if (K % MX_BLOCK) return set_error(MXF8_EINVAL, "%s: K=%lld must be a multiple of 32", what, (long long)K);
  if (M > 0x7fffffff / 2 || K > (1 << 22) || !grid_fits(mx_blocks(M, K), 256))
    return set_error(MXF8_EINVAL, "%s: shape too large", what);
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
  const bool small = mx_small(M, K);
  const dim3 grid((unsigned)mx_blocks(M, K));
  switch (dtype) {
#define MXF8_CASE(DT)                                                                                           \
  case DT:                                                                                                      \
    if (small)                                                                                                  \
      mxfp4_quant_kernel<DT, 2><<<grid, 256, 0, stream>>>(static_cast<const Elem<DT>::T*>(x), ldx, M, (int)K, codes, scales); \
    else                                                                                                        \
      mxfp4_quant_kernel<DT, 4><<<grid, 256, 0, stream>>>(static_cast<const Elem<DT>::T*>(x), ldx, M, (int)K, codes, scales); \
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
  const bool small = mx_small(M, K);
  const dim3 grid((unsigned)mx_blocks(M, K));
  switch (dtype) {
#define MXF8_CASE(DT)                                                                                            \
  case DT:                                                                                                       \
    if (small)                                                                                                   \
      mxfp4_dequant_kernel<DT, 2><<<grid, 256, 0, stream>>>(codes, scales, M, (int)K, static_cast<Elem<DT>::T*>(out)); \
    else                                                                                                         \
      mxfp4_dequant_kernel<DT, 4><<<grid, 256, 0, stream>>>(codes, scales, M, (int)K, static_cast<Elem<DT>::T*>(out)); \
    break;
    MXF8_CASE(MXF8_BF16)
    MXF8_CASE(MXF8_F16)
    MXF8_CASE(MXF8_F32)
#undef MXF8_CASE
    default: return set_error(MXF8_EINVAL, "mxfp4_dequant: bad dtype %d", dtype);
  }
  return check_launch("mxfp4_dequant");
}
