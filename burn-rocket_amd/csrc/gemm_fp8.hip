// Products of many rows with a block-scaled fp8 weight (e4m3 codes, one f32 scale per 128 × 128 block of the weight and per
// row and 128 values of the activations):
//
//   c[m, n] = Σ_b as[m, b] · ws[n / 128, b] · P_b[m, n],  P_b the product of block b's codes,
//
// summed in f32 in block order.
//
// A workgroup takes BM rows × BN outputs and walks K in stages of 128, one block of both scales a stage: LDS slots are
// filled by buffer→LDS copies one stage ahead, weights in the resident layout as they lie (a fragment is 1 KB in one piece,
// free of bank conflicts), rows of activations with 16-byte chunk c of row r at c ^ ((r >> 1) & 7), and the rows' scales of
// the stage behind them. The weight is the first operand, so that a lane holds 16 outputs of one row: a fold is one product
// of two scales and 16 FMAs per 32 × 32 tile and stage, 64 cycles of the VALU for 128 of the matrix unit. Each tile's fold is
// issued behind the next tile's products, so that the two units run side by side.
#include "fp8.hpp"
#include "kernels.hpp"

namespace {
template <int BM, int BN, int WM, int WN, int STAGES>
struct Fp8Geom {
  static constexpr int NW = WM * WN;
  static constexpr int SLOT = (BM + BN) * 128 + BM * 4;
  static constexpr int SMEM = STAGES * SLOT;
  static_assert(SMEM <= 160 * 1024, "LDS per workgroup");
};
}  // namespace

template <int BM, int BN, int WM, int WN, int STAGES, bool EXACT>
__global__ __launch_bounds__(WM *WN * 64, 2) void gemm_fp8_kernel(const Fp8GemmArgs g, int tiles_m, int tiles_n, int group_m) {
  using G = Fp8Geom<BM, BN, WM, WN, STAGES>;
  constexpr int NW = G::NW, SLOT = G::SLOT;
  constexpr int WTM = BM / WM, WTN = BN / WN, TM = WTM / 32, TN = WTN / 32;
  constexpr int QA = BM / 8, QB = BN / 8, QT = QA + QB;  // 1 KB copies of a stage
  constexpr int CP = QT / NW, SI = BM / 64;              // copies per wave; copies of 64 row scales
  static_assert(CP * NW == QT && SI <= NW && SI * 64 == BM, "copies per wave");
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int lane = lane_id(), col = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  int tm, tn;
  tile_coords(xcd_remap(blockIdx.x, gridDim.x), tiles_m, tiles_n, group_m, tm, tn);
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = tn * BN, KT = g.kt;

  const rsrc_t ra = make_rsrc(g.a + m0 * g.k, (g.m - m0) * g.k);
  const rsrc_t rs = make_rsrc(g.as + m0 * KT, (g.m - m0) * KT * 4);
  // (rows of the layout end on a multiple of 128: blocks past it read zeros)
  const int64_t nblk = ((int64_t)g.n + 127) / 128 * 4;
  const rsrc_t rw = make_rsrc(g.w + (int64_t)(n0 / 32) * KT * 4096, (nblk - n0 / 32) * KT * 4096);

  const int r8 = lane >> 3, p8 = lane & 7;
  const uint32_t ch_even = (uint32_t)((p8 ^ (r8 >> 1)) << 4), ch_odd = (uint32_t)((p8 ^ (4 + (r8 >> 1))) << 4);
  auto issue = [&](int slot, int kt) {
    uint8_t *sb = smem + slot * SLOT;
    const uint32_t k0 = (uint32_t)kt * 128;
    const uint32_t even = k0 + ch_even < (uint32_t)g.k ? (uint32_t)(r8 * g.k) + ch_even : OOB_OFFSET;
    const uint32_t odd = k0 + ch_odd < (uint32_t)g.k ? (uint32_t)(r8 * g.k) + ch_odd : OOB_OFFSET;
#pragma unroll
    for (int i = 0; i < CP; ++i) {
      const int q = wave + i * NW;  // wave-uniform
      // (whole offsets in the vector part: that is what the range check of rows past m and of blocks past n sees)
      if (q < QA)
        bdma16(ra, sb + q * 1024, ((q & 1) ? odd : even) + (uint32_t)(q * 8 * g.k) + k0, 0);
      else
        bdma16(rw, sb + q * 1024, lane * 16 + (uint32_t)((((q - QA) >> 2) * KT + kt) * 4096 + ((q - QA) & 3) * 1024), 0);
    }
    if (wave < SI)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, LDS_PTR(sb + QT * 1024 + wave * 256), 4,
                                               (uint32_t)(((wave * 64 + lane) * KT + kt) * 4), 0, 0, 0);
  };

  // A lane's fragment bytes: the row's chunks 4s + 2h + j, swizzled; the weight block's pieces.
  const int swz = (col >> 1) & 7;
  uint32_t a_off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    a_off[i] = (uint32_t)((wm * WTM + col) * 128 + (((4 * (i >> 1) + 2 * h + (i & 1)) ^ swz) << 4));
  const uint32_t w_off = (uint32_t)(BM * 128 + wn * WTN * 128 + lane * 16);
  const uint32_t s_off = (uint32_t)(QT * 1024 + (wm * WTM + col) * 4);
  const float *ws[TN];
#pragma unroll
  for (int i = 0; i < TN; ++i) ws[i] = g.ws + (int64_t)min((n0 + wn * WTN + i * 32) / 128, (int)(nblk / 4) - 1) * KT;

  floatx16 acc[TN][TM], part[2];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    part[1][r] = 0.f;
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j) acc[i][j][r] = 0.f;
  }
  static_assert((TN * TM) % 2 == 0, "the two product registers alternate over stages too");
  float pend = 0.f;  // scale of the tile whose fold is due
  auto load_w = [&](Fp8Frag<EXACT> &f, const uint8_t *sb, int i) {
    const uint8_t *p = sb + w_off + i * 4096;
    f.set(0, *(const intx4 *)p, *(const intx4 *)(p + 1024));
    f.set(1, *(const intx4 *)(p + 2048), *(const intx4 *)(p + 3072));
  };
  auto stage = [&](int slot, int kt) {
    const uint8_t *sb = smem + slot * SLOT;
    Fp8Frag<EXACT> x[TM], w[2];
    float sa[TM], sw[TN];
#pragma unroll
    for (int i = 0; i < TN; ++i) sw[i] = ws[i][kt];
    load_w(w[0], sb, 0);
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const uint8_t *p = sb + j * 32 * 128;
      x[j].set(0, *(const intx4 *)(p + a_off[0]), *(const intx4 *)(p + a_off[1]));
      x[j].set(1, *(const intx4 *)(p + a_off[2]), *(const intx4 *)(p + a_off[3]));
      sa[j] = *(const float *)(sb + s_off + j * 128);
    }
    static_for<TN>([&](auto i_c) {
      constexpr int i = decltype(i_c)::value;
      if constexpr (i + 1 < TN) load_w(w[(i + 1) & 1], sb, i + 1);
      static_for<TM>([&](auto j_c) {
        constexpr int j = decltype(j_c)::value, u = i * TM + j, prev = (u + TN * TM - 1) % (TN * TM);
        part[u & 1] = fp8_product(w[i & 1], x[j]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          acc[prev / TM][prev % TM][r] = __builtin_fmaf(part[(u & 1) ^ 1][r], pend, acc[prev / TM][prev % TM][r]);
        pend = sa[j] * sw[i];
        __builtin_amdgcn_sched_barrier(0);
      });
    });
  };
  issue(0, 0);
  for (int kt = 0; kt < KT; ++kt) {
    WAIT_VMCNT(0);
    WAIT_LGKMCNT0();
    BARRIER();
    if (kt + 1 < KT) issue((kt + 1) % STAGES, kt + 1);
    stage(kt % STAGES, kt);
  }
  constexpr int last = TN * TM - 1;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[TN - 1][TM - 1][r] = __builtin_fmaf(part[last & 1][r], pend, acc[TN - 1][TM - 1][r]);

  const bool whole = (g.n & 3) == 0;
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int64_t m = m0 + wm * WTM + j * 32 + col;
    if (m >= g.m) continue;
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + wn * WTN + i * 32 + q * 8 + h * 4;
        const float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        fp8_store4(g.c, g.c_dtype, m * g.n + n, v, g.n - n, whole);
      }
  }
}

template <int BM, int BN, int WM, int WN, int STAGES, bool EXACT>
static hipError_t launch_fp8(const Fp8GemmArgs &g, hipStream_t st) {
  using G = Fp8Geom<BM, BN, WM, WN, STAGES>;
  auto kern = gemm_fp8_kernel<BM, BN, WM, WN, STAGES, EXACT>;
  static bool attr_set = false;
  if (!attr_set) {
    hipError_t e = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, G::SMEM);
    if (e != hipSuccess) return e;
    attr_set = true;
  }
  const int tm = (int)((g.m + BM - 1) / BM), tn = (g.n + BN - 1) / BN;
  hipLaunchKernelGGL(kern, dim3((unsigned)tm * tn), dim3(G::NW * 64), G::SMEM, st, g, tm, tn, rk_knob("RK_TILE_GROUP_M", 4));
  return hipGetLastError();
}

hipError_t rk_launch_gemm_fp8(const Fp8GemmArgs &g, bool exact, hipStream_t st) {
  if (exact) return launch_fp8<128, 128, 2, 2, 2, true>(g, st);
  const int64_t big = (int64_t)((g.m + 255) / 256) * ((g.n + 255) / 256);
  if (big >= g.num_cus) return launch_fp8<256, 256, 4, 2, 2, false>(g, st);
  return launch_fp8<128, 128, 2, 2, 2, false>(g, st);
}
