// The K loop that the dense and the expert products of many rows share (gemm_fp8.hip, moe_fp8.hip).
#pragma once

#include "fp8.hpp"

// A workgroup takes BM rows × BN outputs and walks K in stages of 128, one block of both scales a stage. LDS slots are
// filled by buffer→LDS copies a stage ahead: weights in the resident layout as they lie (a fragment is 1 KB in one piece,
// free of bank conflicts), rows of activations with 16-byte chunk c of row r at c ^ ((r >> 1) & 7), and the rows' scales of
// the stage behind them. The weight is the first operand, so that a lane holds 16 outputs of one row: a fold is one product
// of two scales and 16 FMAs per 32 × 32 tile and stage, 64 cycles of the VALU for 128 of the matrix unit. Each tile's fold
// is issued behind the next tile's products, so that the two units run side by side.
template <int BM_, int BN_, int WM_, int WN_, int STAGES_, bool EXACT_>
struct Fp8Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_;
  static constexpr bool EXACT = EXACT_;
  static constexpr int NW = WM * WN, NT = NW * 64;
  static constexpr int WTM = BM / WM, WTN = BN / WN, TM = WTM / 32, TN = WTN / 32;
  static constexpr int QA = BM / 8, QB = BN / 8;  // 1 KB copies of a stage
  static constexpr int CA = QA / NW, CB = QB / NW, SI = BM / 64;  // per wave; copies of 64 row scales
  static constexpr int SLOT = (BM + BN) * 128 + BM * 4;
  static constexpr int SMEM = STAGES * SLOT;
  static_assert(SMEM <= 160 * 1024, "LDS per workgroup");
  static_assert(CA * NW == QA && CB * NW == QB && SI <= NW && SI * 64 == BM, "copies per wave");
  static_assert((TN * TM) % 2 == 0, "the two product registers alternate over stages too");

  floatx16 acc[TN][TM];  // outputs 32·i + 8·(r/4) + 4·(lane/32) + r%4 of row 32·j + lane%32 of the wave's part

  // a: codes, rows k bytes apart, a_bytes in all from a; as: scales, rows KT apart. row_of(r): row of `a` for row r of the
  // tile, or -1 (reads zeros). w: the first of the tile's weight blocks, w_bytes in all; ws(i): scales of the wave's block i.
  // rows: of the tile (a wave without any only copies).
  template <typename RowOf, typename Scales>
  __device__ __forceinline__ void run(uint8_t *smem, const uint8_t *a, int64_t a_bytes, const float *as, int64_t as_bytes,
                                      RowOf row_of, int rows, const uint8_t *w, int64_t w_bytes, Scales ws_of, int k, int KT) {
    const int lane = lane_id(), col = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const rsrc_t ra = make_rsrc(a, a_bytes), rs = make_rsrc(as, as_bytes), rw = make_rsrc(w, w_bytes);
    // Whole offsets go into the vector part of a copy's address: that is what the range check sees.
    const int r8 = lane >> 3, p8 = lane & 7;
    uint32_t off[CA], ch[CA];
#pragma unroll
    for (int i = 0; i < CA; ++i) {
      const int r = (wave + i * NW) * 8 + r8;
      const int64_t src = row_of(r);
      ch[i] = (uint32_t)((p8 ^ ((r >> 1) & 7)) << 4);
      off[i] = src < 0 ? OOB_OFFSET : (uint32_t)(src * k) + ch[i];
    }
    uint32_t soff = OOB_OFFSET;
    if (wave < SI) {
      const int64_t src = row_of(wave * 64 + lane);
      if (src >= 0) soff = (uint32_t)(src * KT * 4);
    }
    auto issue = [&](int slot, int kt) {
      uint8_t *sb = smem + slot * SLOT;
      const uint32_t k0 = (uint32_t)kt * 128;
#pragma unroll
      for (int i = 0; i < CA; ++i)
        bdma16(ra, sb + (wave + i * NW) * 1024, k0 + ch[i] < (uint32_t)k ? off[i] + k0 : OOB_OFFSET, 0);
#pragma unroll
      for (int i = 0; i < CB; ++i) {
        const int q = wave + i * NW;
        bdma16(rw, sb + (QA + q) * 1024, lane * 16 + (uint32_t)(((q >> 2) * KT + kt) * 4096 + (q & 3) * 1024), 0);
      }
      if (wave < SI)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, LDS_PTR(sb + (QA + QB) * 1024 + wave * 256), 4, soff + kt * 4, 0, 0, 0);
    };

    // A lane's fragment bytes: the row's chunks 4s + 2h + j, swizzled; the weight block's pieces.
    const int swz = (col >> 1) & 7;
    uint32_t a_off[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      a_off[i] = (uint32_t)((wm * WTM + col) * 128 + (((4 * (i >> 1) + 2 * h + (i & 1)) ^ swz) << 4));
    const uint32_t w_off = (uint32_t)(BM * 128 + wn * WTN * 128 + lane * 16);
    const uint32_t s_off = (uint32_t)((QA + QB) * 1024 + (wm * WTM + col) * 4);
    const float *ws[TN];
#pragma unroll
    for (int i = 0; i < TN; ++i) ws[i] = ws_of(wn * TN + i);

    floatx16 part[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      part[1][r] = 0.f;
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j][r] = 0.f;
    }
    float pend = 0.f;  // scale of the tile whose fold is due
    auto load_w = [&](Fp8Frag<EXACT> &f, const uint8_t *sb, int i) {
      const uint8_t *p = sb + w_off + i * 4096;
      f.set(0, *(const intx4 *)p, *(const intx4 *)(p + 1024));
      f.set(1, *(const intx4 *)(p + 2048), *(const intx4 *)(p + 3072));
    };
    auto stage = [&](int slot, int kt) {
      const uint8_t *sb = smem + slot * SLOT;
      Fp8Frag<EXACT> x[TM], wf[2];
      float sa[TM], sw[TN];
#pragma unroll
      for (int i = 0; i < TN; ++i) sw[i] = ws[i][kt];
      load_w(wf[0], sb, 0);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const uint8_t *p = sb + j * 32 * 128;
        x[j].set(0, *(const intx4 *)(p + a_off[0]), *(const intx4 *)(p + a_off[1]));
        x[j].set(1, *(const intx4 *)(p + a_off[2]), *(const intx4 *)(p + a_off[3]));
        sa[j] = *(const float *)(sb + s_off + j * 128);
      }
      static_for<TN>([&](auto i_c) {
        constexpr int i = decltype(i_c)::value;
        if constexpr (i + 1 < TN) load_w(wf[(i + 1) & 1], sb, i + 1);
        static_for<TM>([&](auto j_c) {
          constexpr int j = decltype(j_c)::value, u = i * TM + j, prev = (u + TN * TM - 1) % (TN * TM);
          part[u & 1] = fp8_product(wf[i & 1], x[j]);
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
      if (wm * WTM < rows) stage(kt % STAGES, kt);
    }
    constexpr int last = TN * TM - 1;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[TN - 1][TM - 1][r] = __builtin_fmaf(part[last & 1][r], pend, acc[TN - 1][TM - 1][r]);
  }
};
