// Product of two matrices in blocks of 32 four-bit values (mxfp4.h), the 4-bit linear:
//
//   out[m, n] = bf16(act(sum_k a[m, k] w[n, k] + bias[n])),  a, w = codes times their block's power of two
//
// on v_mfma_scale_f32_32x32x64_f8f6f4 in its fp4 form, which applies both block scales itself and runs at twice the
// fp8 rate.  The kernel is the row-scaled FP8 GEMM's (gemm.hip) in shape: C^T = W X^T, persistent workgroups
// over output tiles, K stages of 128 bytes per row copied straight to LDS, one barrier in the middle of a stage.
// A stage now holds 256 elements, eight blocks per row.  Lane group g = lane / 32 of a wave takes blocks 4 g .. 4 g + 3
// of its row, one per instruction: any assignment of K to lanes and instructions gives the same sum as long as
// both operands follow it, and with this one the four scales that a lane needs in a stage are one aligned dword
// of the slab's eight bytes per row, which the instruction picks bytes from.
#include "gemm_common.h"
#include "gemm_mxfp4_ring.h"
#include "mxfp4.h"

namespace mxf8 {

// Scale dwords of one stage: this lane's rows of the W and X tiles, blocks 4 g .. 4 g + 3.
template <class C>
struct MxScales {
  uint32_t w[C::TN], x[C::TM];
  // *this = o, as moves that the compiler cannot fold: it would leave the values where they are and put the
  // loads that follow into `o` elsewhere, to be moved at the end of the stage while they are in flight.
  __device__ __forceinline__ void take(const MxScales& o) {
#pragma unroll
    for (int a = 0; a < C::TN; ++a) asm volatile("v_mov_b32 %0, %1" : "=v"(w[a]) : "v"(o.w[a]));
#pragma unroll
    for (int b = 0; b < C::TM; ++b) asm volatile("v_mov_b32 %0, %1" : "=v"(x[b]) : "v"(o.x[b]));
  }
};

template <class C, int ACT, bool KTAIL>
__global__ __launch_bounds__(C::THREADS) void gemm_mxfp4_kernel(const uint8_t* __restrict__ a4, const uint8_t* __restrict__ w4,
                                                                const uint8_t* __restrict__ sa,
                                                                const uint8_t* __restrict__ sw,
                                                                const uint16_t* __restrict__ bias,
                                                                uint16_t* __restrict__ out, int M, int N, int Kb,
                                                                int64_t ld_out, int tiles_m, int tiles_n, int group_m) {
  constexpr int TM = C::TM, TN = C::TN;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * C::STAGE + C::BN * 4];
  float* const ep_b = reinterpret_cast<float*>(smem + 2 * C::STAGE);  // [BN]

  const int ntiles = tiles_m * tiles_n;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wn = wave / C::WM, wm = wave % C::WM;
  const int wrow0 = wn * (C::BN / C::WN), xrow0 = wm * (C::BM / C::WM);
  const int nk = (Kb + GEMM_BK - 1) / GEMM_BK;
  const int r = lane & 31, g = lane >> 5;
  uint32_t lane_off[2];
#pragma unroll
  for (int par = 0; par < 2; ++par)
    lane_off[par] = (uint32_t)((lane >> 3) * Kb) +
                    (uint32_t)(((lane & 7) ^ lds_swz<GEMM_BK>(8 * par + (lane >> 3))) << 4);
  auto rsrc = [&](const uint8_t* base, int row0, int rows, int span) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)(base + (int64_t)row0 * Kb), 0, min(rows - row0, span) * Kb,
                                             0x00020000);
  };

  int s = blockIdx.x;
  int tm, tn;
  tile_coords(s, tiles_m, tiles_n, group_m, tm, tn);
  __amdgpu_buffer_rsrc_t wrs = rsrc(w4, tn * C::BN, N, C::BN), xrs = rsrc(a4, tm * C::BM, M, C::BM);
  gemm_dma<C>(wrs, xrs, smem, lane_off, Kb, wave, 0);
  int gs = 0;  // global stage counter: stage buffer parity runs on across tiles

  for (; s < ntiles; s += gridDim.x) {
    const int m0 = tm * C::BM, n0 = tn * C::BN;
    // this tile's bias, handed over through LDS after the mainloop
    const float ep_v = bias && (int)threadIdx.x < C::BN && n0 + (int)threadIdx.x < N
                           ? bf16_bits_to_f32(bias[n0 + threadIdx.x]) : 0.0f;
    const int s_next = s + gridDim.x;
    int tm_n = 0, tn_n = 0;
    if (s_next < ntiles) tile_coords(s_next, tiles_m, tiles_n, group_m, tm_n, tn_n);

    // rows past the end read the last row's scales (their products are not stored)
    uint32_t ow[TN], ox[TM];
#pragma unroll
    for (int a = 0; a < TN; ++a) ow[a] = min(wrow0 + 32 * a + r, N - 1 - n0) * MX_SLAB + 4 * g;
#pragma unroll
    for (int b = 0; b < TM; ++b) ox[b] = min(xrow0 + 32 * b + r, M - 1 - m0) * MX_SLAB + 4 * g;
    auto load_scales = [&](int ks, MxScales<C>& sc) {
      // (buffer loads: a uniform base and a 32-bit offset, where plain loads would hold six 64-bit addresses)
      const __amdgpu_buffer_rsrc_t pw = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(sw + ((int64_t)ks * N + n0) * MX_SLAB), 0, C::BN * MX_SLAB, 0x00020000);
      const __amdgpu_buffer_rsrc_t px = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(sa + ((int64_t)ks * M + m0) * MX_SLAB), 0, C::BM * MX_SLAB, 0x00020000);
#pragma unroll
      for (int a = 0; a < TN; ++a) sc.w[a] = __builtin_amdgcn_raw_buffer_load_b32(pw, ow[a], 0, 0);
#pragma unroll
      for (int b = 0; b < TM; ++b) sc.x[b] = __builtin_amdgcn_raw_buffer_load_b32(px, ox[b], 0, 0);
    };
    // Blocks past K in the last stage have zeros for codes; their scale bytes, which may hold anything,
    // become 1 (127), as a NaN there would meet the zeros.
    auto mend_scales = [&](MxScales<C>& sc) {
      const int valid = min(max(((Kb % GEMM_BK) >> 4) - 4 * g, 0), 4);
      const uint32_t keep = valid == 4 ? 0xffffffffu : (1u << (8 * valid)) - 1u;
#pragma unroll
      for (int a = 0; a < TN; ++a) sc.w[a] = (sc.w[a] & keep) | (0x7f7f7f7fu & ~keep);
#pragma unroll
      for (int b = 0; b < TM; ++b) sc.x[b] = (sc.x[b] & keep) | (0x7f7f7f7fu & ~keep);
    };

    v16f acc[TN][TM];
#pragma unroll
    for (int a = 0; a < TN; ++a)
#pragma unroll
      for (int b = 0; b < TM; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.0f;

    auto after_last = [&](uint8_t* dst) {
      if (s_next < ntiles) {
        wrs = rsrc(w4, tn_n * C::BN, N, C::BN);
        xrs = rsrc(a4, tm_n * C::BM, M, C::BM);
        gemm_dma<C>(wrs, xrs, dst, lane_off, Kb, wave, 0);
      }
    };
    // Stage 0 of this tile is in flight into buffer gs & 1.
    MxScales<C> cur_s, nxt_s;
    load_scales(0, cur_s);
    wait_vm0();
    block_barrier();
    if (KTAIL && nk == 1) {
      zero_tail<C>(smem + (gs & 1) * C::STAGE, (Kb % GEMM_BK) >> 4);
      mend_scales(cur_s);
      block_barrier();
    }
    if (nk > 1) {
      load_scales(1, nxt_s);
      gemm_dma<C>(wrs, xrs, smem + ((gs + 1) & 1) * C::STAGE, lane_off, Kb, wave, GEMM_BK);
    } else {
      nxt_s = cur_s;
      after_last(smem + ((gs + 1) & 1) * C::STAGE);
    }
    // A stage is four steps, one block of each lane's four per step.  A step's fragments are read while the
    // step before it runs: W's into the registers of the fragment whose products have just been issued, X's
    // into the other of two sets.  Step 3's are the stage's last reads, so the barrier stands before it.
    v4i af[TN], bf[2][TM];
    {
      const uint8_t* cur = smem + (gs & 1) * C::STAGE;
#pragma unroll
      for (int a = 0; a < TN; ++a) af[a] = mx_frag(cur, wrow0 + 32 * a + r, 4 * g);
#pragma unroll
      for (int b = 0; b < TM; ++b) bf[0][b] = mx_frag(cur + C::BN * GEMM_BK, xrow0 + 32 * b + r, 4 * g);
    }
    auto step = [&](auto t_tag, const uint8_t* from, int chunk, const MxScales<C>& sc) {
      constexpr int T = decltype(t_tag)::value;
#pragma unroll
      for (int b = 0; b < TM; ++b) bf[(T + 1) & 1][b] = mx_frag(from + C::BN * GEMM_BK, xrow0 + 32 * b + r, chunk);
#pragma unroll
      for (int a = 0; a < TN; ++a) {
#pragma unroll
        for (int b = 0; b < TM; ++b) acc[a][b] = mx_mma<T>(af[a], bf[T & 1][b], acc[a][b], sc.w[a], sc.x[b]);
        af[a] = mx_frag(from, wrow0 + 32 * a + r, chunk);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    int ks = 0;
    do {
      uint8_t* cur = smem + (gs & 1) * C::STAGE;
      uint8_t* nxt = smem + ((gs + 1) & 1) * C::STAGE;
      step(std::integral_constant<int, 0>{}, cur, 4 * g + 1, cur_s);
      step(std::integral_constant<int, 1>{}, cur, 4 * g + 2, cur_s);
      step(std::integral_constant<int, 2>{}, cur, 4 * g + 3, cur_s);
      // (products have no side effect, and the compiler would move those above past the barrier to their next use)
#pragma unroll
      for (int a = 0; a < TN; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b) asm volatile("" : "+v"(acc[a][b]));
      // (step 3's scales move out of the way here, where the next stage's have landed: moving those while the
      // ones after them are in flight would wait for these)
      const MxScales<C> step3_s = cur_s;
      if (ks + 1 < nk) {
        wait_vm0();
        block_barrier();
        if (KTAIL && ks + 2 == nk) {
          zero_tail<C>(nxt, (Kb % GEMM_BK) >> 4);
          mend_scales(nxt_s);
          block_barrier();
        }
        cur_s.take(nxt_s);
        if (ks + 2 < nk) {
          load_scales(ks + 2, nxt_s);
          gemm_dma<C>(wrs, xrs, cur, lane_off, Kb, wave, (ks + 2) * GEMM_BK);
        } else {
          after_last(cur);
        }
      }
      // (after the last stage the reads fetch nothing that is used)
      step(std::integral_constant<int, 3>{}, nxt, 4 * g, step3_s);
      ++gs;
    } while (++ks < nk);

    // ---- epilogue: acc[a][b] register i is channel n0 + wrow0 + 32 a + 8 (i / 4) + 4 g + i % 4 of token
    // m0 + xrow0 + 32 b + r
    if ((int)threadIdx.x < C::BN) ep_b[threadIdx.x] = ep_v;
    block_barrier();
    // (the lane index is made opaque here, or the epilogue's addresses, the same for every tile, would be held in
    // registers across the mainloop, where there are none left for them)
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int r = ln & 31, g = ln >> 5;
    auto quad = [&](const v16f& c, int q) { return v4f{c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]}; };
    // Each 32-token round of a wave goes through its own 1 / NW of the last stage's buffer and leaves as 16-byte stores
    // of whole row segments, at any alignment; what a tile at the matrix's edge cuts is stored one by one.
    constexpr int RB = TN * 64, NCH = RB / 16, RPI = 64 / NCH;
    static_assert(32 * RB <= C::STAGE / C::NW, "per-wave staging region");
    uint8_t* const wreg = smem + ((gs + 1) & 1) * C::STAGE + wave * (C::STAGE / C::NW);
    const bool inside = m0 + C::BM <= M && n0 + C::BN <= N;
#pragma unroll
    for (int b = 0; b < TM; ++b) {
#pragma unroll
      for (int a = 0; a < TN; ++a)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<uint2*>(wreg + r * RB + (((4 * a + q) ^ (r & (NCH - 1))) << 4) + 8 * g) =
              mx_out_quad<ACT>(quad(acc[a][b], q), *reinterpret_cast<const v4f*>(ep_b + wrow0 + 32 * a + 8 * q + 4 * g));
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int i = 0; i < 32 / RPI; ++i) {
        const int row = i * RPI + ln / NCH, ch = ln % NCH;
        const uint4 val = *reinterpret_cast<const uint4*>(wreg + row * RB + ((ch ^ (row & (NCH - 1))) << 4));
        const int m = m0 + xrow0 + 32 * b + row, n = n0 + wrow0 + ch * 8;
        if (inside)
          mx_store8<true>(out + (int64_t)m * ld_out + n, val, 8);
        else if (m < M)
          mx_store8<true>(out + (int64_t)m * ld_out + n, val, N - n);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    tm = tm_n;
    tn = tn_n;
  }
}

template <class C, int ACT, bool KTAIL>
static void launch_mxfp4(const uint8_t* a4, const uint8_t* w4, const uint8_t* sa, const uint8_t* sw, const uint16_t* bias,
                         uint16_t* out, int M, int N, int Kb, int64_t ld_out, int cus, hipStream_t st) {
  const int tiles_m = (int)cdiv(M, C::BM), tiles_n = (int)cdiv(N, C::BN), ntiles = tiles_m * tiles_n;
  constexpr int per_cu = (160 * 1024) / (2 * C::STAGE + C::BN * 4);
  int grid = cus * per_cu;
  grid = grid >= 8 ? grid & ~7 : ntiles;
  if (grid > ntiles) grid = ntiles;
  const int group_m = Kb >= 8192 ? 4 : 8;
  gemm_mxfp4_kernel<C, ACT, KTAIL><<<dim3(grid), dim3(C::THREADS), 0, st>>>(a4, w4, sa, sw, bias, out, M, N, Kb, ld_out,
                                                                            tiles_m, tiles_n, group_m);
}

typedef MxRing<32, 64, 1, 2, 6> MxRing32x64;      // 77 KB of LDS: two workgroups per CU
typedef MxRing<64, 64, 2, 2, 4> MxRing64x64;      // 68 KB: two
typedef MxRing<128, 64, 4, 2, 3> MxRing128x64;    // 77 KB: two
typedef MxRing<128, 128, 2, 4, 4> MxRing128x128;  // 136 KB: one

template <class C>
static void launch_mxfp4_ring(int act, const uint8_t* a4, const uint8_t* w4, const uint8_t* sa, const uint8_t* sw,
                              const uint16_t* bias, uint16_t* out, int M, int N, int Kb, int64_t ld_out, hipStream_t st) {
  const int tiles_m = (int)cdiv(M, C::BM), tiles_n = (int)cdiv(N, C::BN);
  const bool ktail = Kb % GEMM_BK != 0;
#define MXF8_CASE(A, T)                                                                                        \
  if (act == A && ktail == T)                                                                                  \
    gemm_mxfp4_ring_kernel<C, A, T><<<dim3(tiles_m * tiles_n), dim3(C::THREADS), 0, st>>>(                     \
        a4, w4, sa, sw, bias, out, M, N, Kb, ld_out, tiles_m, tiles_n);
  MXF8_CASE(MXF8_ACT_NONE, false)
  MXF8_CASE(MXF8_ACT_NONE, true)
  MXF8_CASE(MXF8_ACT_GELU_TANH, false)
  MXF8_CASE(MXF8_ACT_GELU_TANH, true)
#undef MXF8_CASE
}

template <int TM, int NW>
static void launch_mxfp4_rows(int act, const uint8_t* a4, const uint8_t* w4, const uint8_t* sa, const uint8_t* sw,
                              const uint16_t* bias, uint16_t* out, int M, int N, int Kb, int64_t ld_out, hipStream_t st) {
  const dim3 grid((unsigned)cdiv(N, 16), (unsigned)cdiv(M, 16 * TM));
  const bool ktail = Kb % GEMM_BK != 0;
#define MXF8_CASE(A, T)                                                                                                 \
  if (act == A && ktail == T)                                                                                           \
    gemm_mxfp4_rows_kernel<TM, NW, A, T><<<grid, 64 * NW, 0, st>>>(a4, w4, sa, sw, bias, out, M, N, Kb, ld_out);
  MXF8_CASE(MXF8_ACT_NONE, false)
  MXF8_CASE(MXF8_ACT_NONE, true)
  MXF8_CASE(MXF8_ACT_GELU_TANH, false)
  MXF8_CASE(MXF8_ACT_GELU_TANH, true)
#undef MXF8_CASE
}

}  // namespace mxf8

using namespace mxf8;

extern "C" int mxf8_gemm_mxfp4(const uint8_t* a4, const uint8_t* w4, const uint8_t* sa, const uint8_t* sw, const void* bias,
                               int act, void* out, int64_t M, int64_t N, int64_t K, int64_t ld_out, hipStream_t stream) {
  const char* what = "gemm_mxfp4";
  if (M < 0 || N < 0 || K < 0) return set_error(MXF8_EINVAL, "%s: negative shape", what);
  if (M == 0 || N == 0) return MXF8_OK;
  if (K == 0 || K % MX_BLOCK) return set_error(MXF8_EINVAL, "%s: K=%lld must be a positive multiple of 32", what, (long long)K);
  if (!a4 || !w4 || !sa || !sw || !out) return set_error(MXF8_EINVAL, "%s: null pointer", what);
  if (ld_out < N) return set_error(MXF8_EINVAL, "%s: ld_out < N", what);
  if (act != MXF8_ACT_NONE && act != MXF8_ACT_GELU_TANH) return set_error(MXF8_EINVAL, "%s: bad act", what);
  if (M > (1 << 27) || N > (1 << 27) || K > (1 << 22)) return set_error(MXF8_EINVAL, "%s: shape too large", what);
  if (((uintptr_t)a4 % 16) || ((uintptr_t)w4 % 16) || ((uintptr_t)sa % 8) || ((uintptr_t)sw % 8))
    return set_error(MXF8_EINVAL, "%s: codes must be 16-byte and scales 8-byte aligned", what);
  const int cus = device_cus();
  if (cus <= 0) return set_error(MXF8_ELAUNCH, "%s: the device's compute-unit count is unavailable", what);
  const int iM = (int)M, iN = (int)N, Kb = (int)(K / 2);
  if (cdiv(M, 128) * cdiv(N, 128) > 0x7fffffff) return set_error(MXF8_EINVAL, "%s: shape too large", what);
  const uint16_t* b16 = static_cast<const uint16_t*>(bias);
  uint16_t* o16 = static_cast<uint16_t*>(out);
#define MXF8_MX_SMALL(launch)                                                        \
  launch(act, a4, w4, sa, sw, b16, o16, iM, iN, Kb, ld_out, stream);                 \
  return check_launch(what);
  const bool ktail = Kb % GEMM_BK != 0;
  const int pick = mxfp4_pick(M, N, K, cus);
  switch (pick) {
    case MX_ROWS16_4: MXF8_MX_SMALL((launch_mxfp4_rows<1, 4>))
    case MX_ROWS16_8: MXF8_MX_SMALL((launch_mxfp4_rows<1, 8>))
    case MX_ROWS16_16: MXF8_MX_SMALL((launch_mxfp4_rows<1, 16>))
    case MX_ROWS32: MXF8_MX_SMALL((launch_mxfp4_rows<2, 4>))
    case MX_RING_32x64: MXF8_MX_SMALL(launch_mxfp4_ring<MxRing32x64>)
    case MX_RING_64x64: MXF8_MX_SMALL(launch_mxfp4_ring<MxRing64x64>)
    case MX_RING_128x64: MXF8_MX_SMALL(launch_mxfp4_ring<MxRing128x64>)
    case MX_RING_128x128: MXF8_MX_SMALL(launch_mxfp4_ring<MxRing128x128>)
    default: break;
  }
#undef MXF8_MX_SMALL
#define MXF8_MX_CASE(Cfg, A, T)                                                                       \
  if (act == A && ktail == T) {                                                                       \
    launch_mxfp4<Cfg, A, T>(a4, w4, sa, sw, b16, o16, iM, iN, Kb, ld_out, cus, stream);               \
    return check_launch(what);                                                                        \
  }
#define MXF8_MX_CASES(Cfg)                                                                                   \
  MXF8_MX_CASE(Cfg, MXF8_ACT_NONE, false) MXF8_MX_CASE(Cfg, MXF8_ACT_NONE, true)                             \
  MXF8_MX_CASE(Cfg, MXF8_ACT_GELU_TANH, false) MXF8_MX_CASE(Cfg, MXF8_ACT_GELU_TANH, true)
  if (pick == MX_TILE_256) {
    MXF8_MX_CASES(GemmBig)
  } else {
    MXF8_MX_CASES(GemmSmall)
  }
#undef MXF8_MX_CASES
#undef MXF8_MX_CASE
  return set_error(MXF8_EINVAL, "%s: no kernel", what);
}
