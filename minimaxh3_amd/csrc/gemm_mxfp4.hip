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
//
// What bounds it: a stage of a 256 x 256 tile is 2048 cycles of products and takes about 3600, an epilogue 9300 a tile, at
// a clock that the power limit holds at 1.9-1.95 GHz.  No unit is busy throughout (matrix cores 44-55%, the vector unit 25-42%,
// LDS active 28-30% of the cycles); waves wait for a third of them.  Without the output stores of whole tiles 4-8% less
// at K = 3072, 2% at 12288.  20280 tokens, once the clock has settled under load (after an idle spell calls take up to 1.3 times as
// long for some ten milliseconds): 3072 -> 12288 403 us (3800 TFLOP/s; the FP8 GEMM 605) and 441 with GELU (651),
// 12288 -> 3072 371 (4130; 616), 3072 -> 9216 314 (467), 3072 -> 3072 108 (161); 8192^3 257 us, 4270 TFLOP/s (407).
// Measured and not kept: four waves of 128 x 128 (spills), W fragments a step ahead too, a barrier in the middle of a
// stage's products, raised wave priority around them.
#include "gemm_common.h"
#include "gemm_mxfp4_ring.h"
#include "mxfp4.h"

namespace mxf8 {

// Scale dwords of one stage: this lane's rows of the W and X tiles, blocks 4 g .. 4 g + 3.
template <class C>
struct MxScales {
  uint32_t w[C::TN], x[C::TM];
  // *this = o, as moves that the compiler does not fold: it would sink the reads of `o` to their first use.
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
  constexpr int SCALES = (C::BM + C::BN) * MX_SLAB;  // a stage's scales: W rows, then X rows
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * C::STAGE + 2 * SCALES + C::BN * 4];
  uint8_t* const sc_smem = smem + 2 * C::STAGE;
  float* const ep_b = reinterpret_cast<float*>(sc_smem + 2 * SCALES);  // [BN]

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
  int tm_c = tm, tn_c = tn;  // the tile that is being copied
  __amdgpu_buffer_rsrc_t wrs = rsrc(w4, tn * C::BN, N, C::BN), xrs = rsrc(a4, tm * C::BM, M, C::BM);
  // Stage ks of tile (tm, tn), whose operands' buffers wrs and xrs are, into stage buffer `buf`.
  auto copy = [&](int buf, int ks) {
    gemm_dma<C>(wrs, xrs, smem + buf * C::STAGE, lane_off, Kb, wave, ks * GEMM_BK);
    mx_copy_scales<C>(sw + ((int64_t)ks * N + tn_c * C::BN) * MX_SLAB, sa + ((int64_t)ks * M + tm_c * C::BM) * MX_SLAB,
                      min(N - tn_c * C::BN, C::BN), min(M - tm_c * C::BM, C::BM), sc_smem + buf * SCALES, wave, lane);
  };
  copy(0, 0);
  // an epilogue round is 32 tokens of a wave's 32 TN channels, 64 x 16 bytes per store
  constexpr int RB = TN * 64, NCH = RB / 16, RPI = 64 / NCH, STORES = TM * (32 / RPI);
  bool stores_behind = false;
  int gs = 0;  // global stage counter: stage buffer parity runs on across tiles

  for (; s < ntiles; s += gridDim.x) {
    const int m0 = tm * C::BM, n0 = tn * C::BN;
    // this tile's bias, handed over through LDS after the mainloop (an unconditional load from a valid address, which
    // nothing waits for here)
    const uint16_t ep_v = *(bias ? bias + min(n0 + (int)(threadIdx.x % C::BN), N - 1) : reinterpret_cast<const uint16_t*>(sw));
    const int s_next = s + gridDim.x;
    int tm_n = 0, tn_n = 0;
    if (s_next < ntiles) tile_coords(s_next, tiles_m, tiles_n, group_m, tm_n, tn_n);

    v16f acc[TN][TM];
#pragma unroll
    for (int a = 0; a < TN; ++a)
#pragma unroll
      for (int b = 0; b < TM; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.0f;

    // the next tile's first stage
    auto after_last = [&](int buf) {
      if (s_next < ntiles) {
        tm_c = tm_n;
        tn_c = tn_n;
        wrs = rsrc(w4, tn_n * C::BN, N, C::BN);
        xrs = rsrc(a4, tm_n * C::BM, M, C::BM);
        copy(buf, 0);
      }
    };
    // Blocks past K in the last stage: zero codes, and scales of 1 (127) in the place of bytes that may hold anything
    // (a NaN would meet the zeros).
    auto mend = [&](int buf) {
      const int valid = (Kb % GEMM_BK) >> 4;
      zero_tail<C>(smem + buf * C::STAGE, valid);
      for (int i = threadIdx.x; i < SCALES; i += C::THREADS)
        if (i % MX_SLAB >= valid) sc_smem[buf * SCALES + i] = 127;
      block_barrier();
    };
    // Stage 0 of this tile is in flight into buffer gs & 1; the last tile's output stores (STORES a wave, of a tile
    // inside the matrix), issued after it, are not waited for.  The bias load is not counted: the compiler may place it
    // on either side of the wait, and one operation too many here would leave a copy in flight.
    if (stores_behind)
      wait_vm<STORES>();
    else
      wait_vm0();
    block_barrier();
    if (KTAIL && nk == 1) mend(gs & 1);
    if (nk > 1)
      copy((gs + 1) & 1, 1);
    else
      after_last((gs + 1) & 1);
    // A stage is four steps, one block of each lane's four per step.  A step's fragments are read while the
    // step before it runs: W's into the registers of the fragment whose products have just been issued, X's
    // into the other of two sets.  Step 3's are the stage's last reads, so the barrier stands before it.
    v4i af[TN], bf[2][TM];
    MxScales<C> sc, sc_next;
    auto read_scales = [&](int buf, MxScales<C>& to) {
      const uint8_t* p = sc_smem + buf * SCALES + 4 * g;
#pragma unroll
      for (int a = 0; a < TN; ++a) to.w[a] = *reinterpret_cast<const uint32_t*>(p + (wrow0 + 32 * a + r) * MX_SLAB);
#pragma unroll
      for (int b = 0; b < TM; ++b)
        to.x[b] = *reinterpret_cast<const uint32_t*>(p + (C::BN + xrow0 + 32 * b + r) * MX_SLAB);
    };
    {
      const uint8_t* cur = smem + (gs & 1) * C::STAGE;
#pragma unroll
      for (int a = 0; a < TN; ++a) af[a] = mx_frag(cur, wrow0 + 32 * a + r, 4 * g);
#pragma unroll
      for (int b = 0; b < TM; ++b) bf[0][b] = mx_frag(cur + C::BN * GEMM_BK, xrow0 + 32 * b + r, 4 * g);
      read_scales(gs & 1, sc);
    }
    auto step = [&](auto t_tag, const uint8_t* from, int chunk) {
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
      const int cb = gs & 1, nb = cb ^ 1;
      uint8_t* cur = smem + cb * C::STAGE;
      uint8_t* nxt = smem + nb * C::STAGE;
      step(std::integral_constant<int, 0>{}, cur, 4 * g + 1);
      step(std::integral_constant<int, 1>{}, cur, 4 * g + 2);
      step(std::integral_constant<int, 2>{}, cur, 4 * g + 3);
      // (products have no side effect, and the compiler would move those above past the barrier to their next use)
#pragma unroll
      for (int a = 0; a < TN; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b) asm volatile("" : "+v"(acc[a][b]));
      if (ks + 1 < nk) {
        wait_vm0();
        block_barrier();
        if (KTAIL && ks + 2 == nk) mend(nb);
        if (ks + 2 < nk)
          copy(cb, ks + 2);
        else
          after_last(cb);
      }
      // (after the last stage the reads fetch nothing that is used)
      read_scales(nb, sc_next);
      step(std::integral_constant<int, 3>{}, nxt, 4 * g);
      sc.take(sc_next);
      ++gs;
    } while (++ks < nk);

    // ---- epilogue: acc[a][b] register i is channel n0 + wrow0 + 32 a + 8 (i / 4) + 4 g + i % 4 of token
    // m0 + xrow0 + 32 b + r
    if ((int)threadIdx.x < C::BN) ep_b[threadIdx.x] = bias ? bf16_bits_to_f32(ep_v) : 0.0f;
    block_barrier();
    // (the lane index is made opaque here, or the epilogue's addresses, the same for every tile, would be held in
    // registers across the mainloop, where there are none left for them)
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int r = ln & 31, g = ln >> 5;
    auto quad = [&](const v16f& c, int q) { return v4f{c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]}; };
    // Each 32-token round of a wave goes through its own 1 / NW of the last stage's buffer and leaves as 16-byte stores
    // of whole row segments, at any alignment; what a tile at the matrix's edge cuts is stored one by one.
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
    stores_behind = inside;
    tm = tm_n;
    tn = tn_n;
  }
}

template <class C, int ACT, bool KTAIL>
static void launch_mxfp4(const uint8_t* a4, const uint8_t* w4, const uint8_t* sa, const uint8_t* sw, const uint16_t* bias,
                         uint16_t* out, int M, int N, int Kb, int64_t ld_out, int cus, hipStream_t st) {
  const int tiles_m = (int)cdiv(M, C::BM), tiles_n = (int)cdiv(N, C::BN), ntiles = tiles_m * tiles_n;
  constexpr int per_cu = (160 * 1024) / (2 * C::STAGE + 2 * (C::BM + C::BN) * MX_SLAB + C::BN * 4);
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

template <int TM, int TN, int NW, int XT>
static void launch_mxfp4_rows(int act, const void* x, int64_t ldx, const uint8_t* sa, const uint8_t* w4, const uint8_t* sw,
                              const uint16_t* bias, uint16_t* out, int M, int N, int Kb, int64_t ld_out, hipStream_t st) {
  const dim3 grid((unsigned)cdiv(N, 16 * TN), (unsigned)cdiv(M, 16 * TM));
  const int lds = XT == MX_CODES ? 0 : M * mx_row_pitch((int)cdiv(Kb, GEMM_BK));
  const bool ktail = Kb % GEMM_BK != 0;
#define MXF8_CASE(A, T)                                                                                             \
  if (act == A && ktail == T)                                                                                       \
    gemm_mxfp4_rows_kernel<TM, TN, NW, A, T, XT><<<grid, 64 * NW, lds, st>>>(x, ldx, sa, w4, sw, bias, out, M, N, Kb, ld_out);
  MXF8_CASE(MXF8_ACT_NONE, false)
  MXF8_CASE(MXF8_ACT_NONE, true)
  MXF8_CASE(MXF8_ACT_GELU_TANH, false)
  MXF8_CASE(MXF8_ACT_GELU_TANH, true)
#undef MXF8_CASE
}

// The rows kernel that mxfp4_pick chose.
template <int XT>
static void launch_mxfp4_few(int pick, int act, const void* x, int64_t ldx, const uint8_t* sa, const uint8_t* w4,
                             const uint8_t* sw, const uint16_t* bias, uint16_t* out, int M, int N, int Kb, int64_t ld_out,
                             hipStream_t st) {
#define MXF8_ROWS(TM, TN, NW) \
  launch_mxfp4_rows<TM, TN, NW, XT>(act, x, ldx, sa, w4, sw, bias, out, M, N, Kb, ld_out, st)
  switch (pick) {
    case MX_ROWS16_4: MXF8_ROWS(1, 1, 4); break;
    case MX_ROWS16_8: MXF8_ROWS(1, 1, 8); break;
    case MX_ROWS16_16: MXF8_ROWS(1, 1, 16); break;
    case MX_ROWS32x32:
      if constexpr (XT == MX_CODES) MXF8_ROWS(2, 2, 8);
      break;
    default:
      if constexpr (XT == MX_CODES) MXF8_ROWS(2, 1, 8);
  }
#undef MXF8_ROWS
}

// Checks of the product that its two entries share.
static int mxfp4_check(const char* what, const uint8_t* w4, const uint8_t* sw, int act, const void* out, int64_t M, int64_t N,
                       int64_t K, int64_t ld_out) {
  if (K <= 0 || K % MX_BLOCK) return set_error(MXF8_EINVAL, "%s: K=%lld must be a positive multiple of 32", what, (long long)K);
  if (!w4 || !sw || !out) return set_error(MXF8_EINVAL, "%s: null pointer", what);
  if (ld_out < N) return set_error(MXF8_EINVAL, "%s: ld_out < N", what);
  if (act != MXF8_ACT_NONE && act != MXF8_ACT_GELU_TANH) return set_error(MXF8_EINVAL, "%s: bad act", what);
  if (M > (1 << 27) || N > (1 << 27) || K > (1 << 22) || cdiv(M, 32) * cdiv(N, 64) > 0x7fffffff)
    return set_error(MXF8_EINVAL, "%s: shape too large", what);
  if (((uintptr_t)w4 % 16) || ((uintptr_t)sw % 8))
    return set_error(MXF8_EINVAL, "%s: codes must be 16-byte and scales 8-byte aligned", what);
  return MXF8_OK;
}

}  // namespace mxf8

using namespace mxf8;

extern "C" int mxf8_gemm_mxfp4(const uint8_t* a4, const uint8_t* w4, const uint8_t* sa, const uint8_t* sw, const void* bias,
                               int act, void* out, int64_t M, int64_t N, int64_t K, int64_t ld_out, hipStream_t stream) {
  const char* what = "gemm_mxfp4";
  if (M < 0 || N < 0 || K < 0) return set_error(MXF8_EINVAL, "%s: negative shape", what);
  if (M == 0 || N == 0) return MXF8_OK;
  if (const int rc = mxfp4_check(what, w4, sw, act, out, M, N, K, ld_out)) return rc;
  if (!a4 || !sa) return set_error(MXF8_EINVAL, "%s: null pointer", what);
  if (((uintptr_t)a4 % 16) || ((uintptr_t)sa % 8))
    return set_error(MXF8_EINVAL, "%s: codes must be 16-byte and scales 8-byte aligned", what);
  const int cus = device_cus();
  if (cus <= 0) return set_error(MXF8_ELAUNCH, "%s: the device's compute-unit count is unavailable", what);
  const int iM = (int)M, iN = (int)N, Kb = (int)(K / 2);
  const uint16_t* b16 = static_cast<const uint16_t*>(bias);
  uint16_t* o16 = static_cast<uint16_t*>(out);
  const bool ktail = Kb % GEMM_BK != 0;
  const int pick = mxfp4_pick(M, N, K, cus);
#define MXF8_MX_RING(Cfg)                                                                             \
  launch_mxfp4_ring<Cfg>(act, a4, w4, sa, sw, b16, o16, iM, iN, Kb, ld_out, stream);                  \
  break;
#define MXF8_MX_CASE(Cfg, A, T) \
  if (act == A && ktail == T) launch_mxfp4<Cfg, A, T>(a4, w4, sa, sw, b16, o16, iM, iN, Kb, ld_out, cus, stream);
#define MXF8_MX_TILE(Cfg)                                                                             \
  MXF8_MX_CASE(Cfg, MXF8_ACT_NONE, false)                                                             \
  MXF8_MX_CASE(Cfg, MXF8_ACT_NONE, true)                                                              \
  MXF8_MX_CASE(Cfg, MXF8_ACT_GELU_TANH, false)                                                        \
  MXF8_MX_CASE(Cfg, MXF8_ACT_GELU_TANH, true)                                                         \
  break;
  switch (pick) {
    case MX_RING_32x64: MXF8_MX_RING(MxRing32x64)
    case MX_RING_64x64: MXF8_MX_RING(MxRing64x64)
    case MX_RING_128x64: MXF8_MX_RING(MxRing128x64)
    case MX_RING_128x128: MXF8_MX_RING(MxRing128x128)
    case MX_TILE_128: MXF8_MX_TILE(GemmSmall)
    case MX_TILE_256: MXF8_MX_TILE(GemmBig)
    default: launch_mxfp4_few<MX_CODES>(pick, act, a4, 0, sa, w4, sw, b16, o16, iM, iN, Kb, ld_out, stream);
  }
#undef MXF8_MX_TILE
#undef MXF8_MX_CASE
#undef MXF8_MX_RING
  return check_launch(what);
}

// Whether the product quantizes its activations itself: the rows kernel's tokens, in 16 bits, as long as what every
// workgroup spends on it (M K elements, the first of them while the weights are on their way) is less than the launch
// it saves (and the host a launch).  With more than one workgroup per compute unit the limit is lower.  MI355X, one
// launch / two, in a graph: 1 x 3072 x 3072 3.5 / 5.2 us, 16 x 3072 x 3072 5.1 / 6.2, 1 x 9216 x 3072 6.4 / 8.3,
// 8 x 9216 x 3072 8.9 / 9.8, 1 x 3072 x 12288 7.7 / 9.6, 1 x 12288 x 12288 16.6 / 19.3; past the limits
// 12 x 9216 x 3072 10.6 / 9.7, 16 x 3072 x 6144 8.6 / 8.3.
static bool mxfp4_one_launch(int64_t M, int64_t N, int64_t K, int dtype) {
  return M <= 16 && dtype != MXF8_F32 && M * K <= (N > 4096 ? 32768 : 65536);
}

extern "C" int64_t mxf8_mxfp4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype) {
  if (M <= 0 || N <= 0 || K <= 0 || N > (1 << 27) || K > (1 << 22) || mxfp4_one_launch(M, N, K, dtype)) return 0;
  return M * (K / 2) + mx_slabs(K) * M * MX_SLAB;  // codes, then scales (K / 2 is a multiple of 16)
}

extern "C" int mxf8_mxfp4_linear(const void* x, int dtype, int64_t ldx, const uint8_t* w4, const uint8_t* sw, const void* bias,
                                 int act, void* out, int64_t M, int64_t N, int64_t K, int64_t ld_out, void* workspace,
                                 hipStream_t stream) {
  const char* what = "mxfp4_linear";
  if (M < 0 || N < 0 || K < 0) return set_error(MXF8_EINVAL, "%s: negative shape", what);
  if (M == 0 || N == 0) return MXF8_OK;
  if (const int rc = mxfp4_check(what, w4, sw, act, out, M, N, K, ld_out)) return rc;
  if (!x) return set_error(MXF8_EINVAL, "%s: null pointer", what);
  if (ldx < K && M > 1) return set_error(MXF8_EINVAL, "%s: ldx < K", what);
  if (dtype != MXF8_BF16 && dtype != MXF8_F16 && dtype != MXF8_F32)
    return set_error(MXF8_EINVAL, "%s: bad dtype %d", what, dtype);
  if (!mxfp4_one_launch(M, N, K, dtype)) {
    if (!workspace || (uintptr_t)workspace % 16) return set_error(MXF8_EINVAL, "%s: a 16-byte aligned workspace is needed", what);
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    uint8_t* scales = codes + M * (K / 2);
    if (const int rc = mxf8_mxfp4_quant(x, dtype, M, K, ldx, codes, scales, stream)) return rc;
    return mxf8_gemm_mxfp4(codes, w4, scales, sw, bias, act, out, M, N, K, ld_out, stream);
  }
  const int cus = device_cus();
  if (cus <= 0) return set_error(MXF8_ELAUNCH, "%s: the device's compute-unit count is unavailable", what);
  const int pick = mxfp4_pick(M, N, K, cus);  // a rows kernel
  const uint16_t* b16 = static_cast<const uint16_t*>(bias);
  uint16_t* o16 = static_cast<uint16_t*>(out);
#define MXF8_CASE(DT)                                                                                                 \
  if (dtype == DT)                                                                                                    \
    launch_mxfp4_few<DT>(pick, act, x, ldx, nullptr, w4, sw, b16, o16, (int)M, (int)N, (int)(K / 2), ld_out, stream);
  MXF8_CASE(MXF8_BF16)
  MXF8_CASE(MXF8_F16)
#undef MXF8_CASE
  return check_launch(what);
}
