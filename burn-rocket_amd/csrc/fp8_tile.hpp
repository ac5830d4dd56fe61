// The K loops of the dense and the expert products of many rows (gemm_fp8.hip, moe_fp8.hip).
#pragma once

#include "fp8.hpp"

// The thread's index as a new value: what an epilogue computes from it is not kept in registers through the K loop.
__device__ __forceinline__ int fresh_tid() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// A workgroup takes BM rows × BN outputs and walks K in stages of 128, one block of both scales a stage. LDS slots are
// filled by buffer→LDS copies a stage ahead: weights in the resident layout as they lie (a fragment is 1 KB in one piece,
// free of bank conflicts), rows of activations with 16-byte chunk c of row r at c ^ ((r >> 1) & 7), and the rows' scales of
// the stage and the blocks' behind them. The weight is the first operand, so that a lane holds 16 outputs of one row: a fold
// is one product of two scales and 16 FMAs per 32 × 32 tile and stage, 64 cycles of the VALU for 128 of the matrix unit;
// a SIMD's other wave has the matrix unit meanwhile. The barrier of a stage stands before its last row of tiles: by then its
// fragments are in registers, so its slot is refilled and the next stage's first fragments are read under that row's
// products.
//
// 16000 × 4096 × 4096 on MI355X, 256 × 256: 244 us, 2.2 PFLOP/s. Without the folds as much, without the copies 214, without
// these and the stores 197. Tried: folds a tile behind in a second set of product registers (spills; 302 with fewer other
// registers kept); the copies in one go behind the barrier (274) or all in the last row (265).
template <int BM_, int BN_, int WM_, int WN_, int STAGES_, bool EXACT_>
struct Fp8Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_;
  static constexpr bool EXACT = EXACT_;
  static constexpr int NW = WM * WN, NT = NW * 64;
  static constexpr int WTM = BM / WM, WTN = BN / WN, TM = WTM / 32, TN = WTN / 32;
  static constexpr int QA = BM / 8, QB = BN / 8;  // 1 KB copies of a stage
  static constexpr int CA = QA / NW, CB = QB / NW, SI = BM / 64;  // per wave; copies of 64 row scales
  static constexpr int WS_AT = (BM + BN) * 128 + BM * 4;  // the weight blocks' scales, [BN / 32]
  static constexpr int SLOT = WS_AT + 256;
  static constexpr int SMEM = STAGES * SLOT;
  static_assert(SMEM <= 160 * 1024, "LDS per workgroup");
  static_assert(CA * NW == QA && CB * NW == QB && SI < NW && SI * 64 == BM, "copies per wave");
  static_assert((TN * TM) % 2 == 0 && TN % 2 == 0, "the two product registers and the two weight fragments alternate over stages too");
  static_assert(STAGES >= 2, "the slot of a stage is refilled for the one STAGES later");

  floatx16 acc[TN][TM];  // outputs 32·i + 8·(r/4) + 4·(lane/32) + r%4 of row 32·j + lane%32 of the wave's part

  // a: codes, rows k bytes apart, a_bytes in all from a; as: scales, rows KT apart. row_of(r): row of `a` for row r of the
  // tile, or -1 (reads zeros). w: the tile's weight blocks, as many as there are (a block past them
  // reads the last one: its results are not stored); ws_of(i): of the scales `ws` (ws_bytes), the first one of the
  // workgroup's block i. rows: of the tile (a wave without any only copies).
  template <typename RowOf, typename Scales>
  __device__ __forceinline__ void run(uint8_t *smem, const uint8_t *a, int64_t a_bytes, const float *as, int64_t as_bytes,
                                      RowOf row_of, int rows, const uint8_t *w, int blocks, const float *ws, int64_t ws_bytes,
                                      Scales ws_of, int k, int KT) {
    const int lane = lane_id(), col = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const rsrc_t ra = make_rsrc(a, a_bytes), rw = make_rsrc(w, (int64_t)min(blocks, BN / 32) * KT * 4096);
    // Rows past the tile's and lanes past K have vector offsets that every range check refuses; what the scalar part adds
    // to the others stays inside a row, or inside the weight's blocks.
    const int r8 = lane >> 3, p8 = lane & 7;
    static_assert(NW % 2 == 0, "a wave's copies share their chunks' order");
    const uint32_t ch = (uint32_t)((p8 ^ (((wave * 8 + r8) >> 1) & 7)) << 4);
    uint32_t off[CA];
#pragma unroll
    for (int i = 0; i < CA; ++i) {
      const int64_t src = row_of((wave + i * NW) * 8 + r8);
      off[i] = src < 0 ? OOB_OFFSET : (uint32_t)(src * k) + ch;
    }
    // One copy of scales a wave: of 64 rows, or (all others, to the same place) of the weight blocks.
    const bool row_scales = wave < SI;
    const rsrc_t rsc = row_scales ? make_rsrc(as, as_bytes) : make_rsrc(ws, ws_bytes);
    const int sc_at = row_scales ? (QA + QB) * 1024 + wave * 256 : WS_AT;
    uint32_t soff = OOB_OFFSET;
    if (row_scales) {
      const int64_t src = row_of(wave * 64 + lane);
      if (src >= 0) soff = (uint32_t)(src * KT * 4);
    } else if (lane < BN / 32) {
      soff = (uint32_t)(ws_of(lane) * 4);
    }
    // Copies [FROM, TO) of a stage.
    constexpr int CP = CA + CB + 1;
    auto issue = [&](auto from_c, auto to_c, int slot, int kt) {
      uint8_t *sb = smem + slot * SLOT;
      const uint32_t k0 = (uint32_t)kt * 128;
      static_for<decltype(to_c)::value - decltype(from_c)::value>([&](auto c_c) {
        constexpr int c = decltype(c_c)::value + decltype(from_c)::value;
        if constexpr (c < CA) {
          bdma16(ra, sb + (wave + c * NW) * 1024, k0 + ch < (uint32_t)k ? off[c] : OOB_OFFSET, k0);
        } else if constexpr (c < CA + CB) {
          const int q = wave + (c - CA) * NW;
          bdma16(rw, sb + (QA + q) * 1024, lane * 16, (uint32_t)((min(q >> 2, blocks - 1) * KT + kt) * 4096 + (q & 3) * 1024));
        } else {
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rsc, LDS_PTR(sb + sc_at), 4, soff, kt * 4, 0, 0);
        }
      });
    };
    // A stage's copies are dealt out over the tiles behind the barrier that frees their slot: the last row of tiles, and the
    // next stage's first one if that leaves them a row's time to arrive. In one go they hold the waves up for a fifth of a
    // stage (72 copies of 64 lanes through one address unit).
    constexpr int SPREAD = TN > 2 ? 2 * TM : TM, QUOTA = (CP + SPREAD - 1) / SPREAD;
    auto issue_at = [&](auto step_c, int slot, int kt) {
      constexpr int f = decltype(step_c)::value * QUOTA, t = f + QUOTA;
      if constexpr (decltype(step_c)::value < SPREAD && f < CP) issue(ic<f>{}, ic<(t < CP ? t : CP)>{}, slot, kt);
    };

    // A lane's fragment bytes: the row's chunks 4s + 2h + j, swizzled; the weight block's pieces.
    const int swz = (col >> 1) & 7;
    const uint32_t a_off = (uint32_t)((wm * WTM + col) * 128 + (((2 * h) ^ swz) << 4));  // (chunk bits 0 and 2: ^ 16, ^ 64)
    const uint32_t w_off = (uint32_t)(BM * 128 + wn * WTN * 128 + lane * 16);
    const uint32_t s_off = (uint32_t)((QA + QB) * 1024 + (wm * WTM + col) * 4);

#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j][r] = 0.f;
    Fp8Frag<EXACT> x[TM], wf[2];
    float sa[TM], sw[TN];
    auto load_w = [&](Fp8Frag<EXACT> &f, int slot, int i) {
      const uint8_t *p = smem + slot * SLOT + w_off + i * 4096;
      f.set(0, *(const intx4 *)p, *(const intx4 *)(p + 1024));
      f.set(1, *(const intx4 *)(p + 2048), *(const intx4 *)(p + 3 * 1024));
    };
    auto load_x = [&](int slot, int j) {
      const uint8_t *p = smem + slot * SLOT + j * 32 * 128;
      x[j].set(0, *(const intx4 *)(p + a_off), *(const intx4 *)(p + (a_off ^ 16)));
      x[j].set(1, *(const intx4 *)(p + (a_off ^ 64)), *(const intx4 *)(p + (a_off ^ 80)));
    };
    // (the scales of the last row of tiles are used up before the next stage's are read)
    auto load_s = [&](int slot) {
#pragma unroll
      for (int j = 0; j < TM; ++j) sa[j] = *(const float *)(smem + slot * SLOT + s_off + j * 128);
#pragma unroll
      for (int i = 0; i < TN; ++i) sw[i] = *(const float *)(smem + slot * SLOT + WS_AT + (wn * TN + i) * 4);
    };
    auto tile = [&](auto i_c, auto j_c) {
      constexpr int i = decltype(i_c)::value, j = decltype(j_c)::value;
      const floatx16 p = fp8_half(wf[i & 1], x[j], 1, fp8_half(wf[i & 1], x[j], 0, floatx16{}));
      const float sc = sa[j] * sw[i];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = __builtin_fmaf(p[r], sc, acc[i][j][r]);
      __builtin_amdgcn_sched_barrier(0);
    };
    // The copies of a wave's next stage have arrived when those of the `behind` ones after it are left (every wave issues CP a stage).
    auto arrived = [&](auto behind_c) {
      WAIT_VMCNT(decltype(behind_c)::value * CP);
      WAIT_LGKMCNT0();
      BARRIER();
    };
    constexpr int AHEAD = STAGES - 2;  // stages in flight at a barrier behind the one that it waits for
    static_assert(AHEAD * CP < 64, "copies that the wait can count");
    const int pre = min(KT, STAGES - 1);
    for (int kt = 0; kt < pre; ++kt) issue(ic<0>{}, ic<CP>{}, kt, kt);
    if (KT > AHEAD) arrived(ic<AHEAD>{});
    else arrived(ic<0>{});
    auto after = [](int slot, int by) { return slot + by >= STAGES ? slot + by - STAGES : slot + by; };
    int slot = 0;
    if (wm * WTM >= rows) {  // a wave without rows copies for the others
      for (int kt = 0; kt + 1 < KT; ++kt, slot = after(slot, 1)) {
        if (kt + STAGES - 1 < KT) {
          issue(ic<0>{}, ic<CP>{}, after(slot, STAGES - 1), kt + STAGES - 1);
          arrived(ic<AHEAD>{});
        } else {
          arrived(ic<0>{});
        }
      }
    } else {
      load_w(wf[0], 0, 0);
#pragma unroll
      for (int j = 0; j < TM; ++j) load_x(0, j);
      load_s(0);
      if (KT >= STAGES) static_for<TM>([&](auto j_c) { issue_at(j_c, STAGES - 1, STAGES - 1); });
      // more: a stage follows; last: the stage STAGES - 1 later exists; most: the one STAGES later too (no branches in the steady state)
      auto stage = [&](int kt, auto more_c, auto last_c, auto most_c) {
        constexpr bool more = decltype(more_c)::value, last = decltype(last_c)::value, most = decltype(most_c)::value;
        const int next = after(slot, 1);
        static_for<TN - 1>([&](auto i_c) {
          load_w(wf[(decltype(i_c)::value + 1) & 1], slot, decltype(i_c)::value + 1);
          static_for<TM>([&](auto j_c) {
            tile(i_c, j_c);
            if constexpr (last && decltype(i_c)::value == 0) issue_at(ic<TM + decltype(j_c)::value>{}, after(slot, STAGES - 1), kt + STAGES - 1);
          });
        });
        if constexpr (more) {
          arrived(ic<last ? AHEAD : 0>{});
          load_w(wf[0], next, 0);
        }
        static_for<TM>([&](auto j_c) {
          tile(ic<TN - 1>{}, j_c);
          if constexpr (most) issue_at(j_c, slot, kt + STAGES);
          if constexpr (more) load_x(next, decltype(j_c)::value);
        });
        if constexpr (more) load_s(next);
        slot = next;
      };
      int kt = 0;
      for (; kt + STAGES < KT; ++kt) stage(kt, ic<1>{}, ic<1>{}, ic<1>{});
      if (kt + STAGES == KT) stage(kt++, ic<1>{}, ic<1>{}, ic<0>{});
      for (; kt + 1 < KT; ++kt) stage(kt, ic<1>{}, ic<0>{}, ic<0>{});
      stage(kt, ic<0>{}, ic<0>{}, ic<0>{});
    }
    __syncthreads();  // the slots may be used for something else
  }
};

// The tile's results to rows of a matrix through LDS, so that a wave stores whole pieces of a row (its lanes hold four
// outputs of 32 rows each: 16-byte pieces of 32 lines, which cost a third of the vision layer's 4304 × 1152 product).
// value(i, j, r): the lane's result; to: the tile's first row, ld values apart; n: outputs from the tile's first on.
// Chunk c of 16 bytes of row r lies at c ^ (r mod 32) (16 of a narrow row): the rows that a store writes are on different banks.
template <class T, int DT, typename Value>
__device__ __forceinline__ void fp8_store_tile(uint8_t *smem, Value value, void *to, int64_t ld, int rows, int n) {
  constexpr int BM = T::BM, BN = T::BN, WN = T::WN, WTM = T::WTM, WTN = T::WTN, TM = T::TM, TN = T::TN, NT = T::NT;
  constexpr int ES = DT == RK_DTYPE_F32 ? 4 : 2, V = 16 / ES;  // values of a chunk
  constexpr int ROWB = BN * ES, CH = ROWB / 16;                 // a row's bytes and chunks
  constexpr int SW = CH < 32 ? CH - 1 : 31;
  static_assert(BM * ROWB <= T::SMEM && (CH & (CH - 1)) == 0 && NT % CH == 0, "the tile in LDS");
  const int tid = fresh_tid(), col = tid & 31, h = (tid >> 5) & 1;
  const int wave = tid >> 6, wm = wave / WN, wn = wave % WN;
#pragma unroll
  for (int j = 0; j < TM; ++j)
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float v[4] = {value(i, j, 4 * q), value(i, j, 4 * q + 1), value(i, j, 4 * q + 2), value(i, j, 4 * q + 3)};
        const int r = wm * WTM + j * 32 + col, at = wn * WTN + i * 32 + q * 8 + h * 4;
        fp8_encode4<DT>(smem + r * ROWB + (((at / V) ^ (r & SW)) * 16) + at % V * ES, v);
      }
  __syncthreads();
  const int c = tid % CH, left = n - c * V;
  if (left <= 0) return;
  // (gfx950 stores 16 bytes at any address; a row of an odd length begins between two of its pieces. 3536 rows of 6780 at
  // K = 384 value by value: 42 us instead of 22)
  typedef uint32_t piece __attribute__((ext_vector_type(4), aligned(2)));
  const bool whole = left >= V;
  for (int r = tid / CH; r < rows; r += NT / CH) {
    const uint8_t *p = smem + r * ROWB + ((c ^ (r & SW)) * 16);
    uint8_t *o = (uint8_t *)to + (r * ld + c * V) * ES;
    if (whole) {
      *(piece *)o = *(const uintx4 *)p;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < left) ((dt_storage<DT> *)o)[e] = ((const dt_storage<DT> *)p)[e];
    }
  }
}

// Smaller tiles, with the weights' fragments straight from memory to registers, as they lie: four waves of all BM rows and 32
// outputs each, so that no two ask for the same weights, and LDS, which bounds such tiles otherwise, holds the rows alone.
// STAGES - 1 stages of both are on the way. A stage of 64 × 128 takes 0.36 us of
// its CU on MI355X, of two tiles there 0.54 both (products 0.12 and 0.24, the 24 KB of each 0.2 at what a CU reads out of its L2):
// barrier, LDS, products and folds one behind the other, which three stages or four, or K split over two groups of waves,
// change little.
template <int TM_, int STAGES_, bool EXACT_>
struct Fp8Flow {
  static constexpr int TM = TM_, TN = 1, STAGES = STAGES_, WM = 1, WN = 4, NW = 4, NT = 256;
  static constexpr bool EXACT = EXACT_;
  static constexpr int BM = 32 * TM, BN = 128 * TN, WTM = BM, WTN = 32 * TN;
  static constexpr int QA = BM / 8, CA = QA / NW, SI = BM / 64;
  static constexpr int WS_AT = BM * 128 + BM * 4;
  static constexpr int SLOT = WS_AT + 256;
  static constexpr int OUT = BM * BN * (EXACT ? 4 : 2);
  static constexpr int SMEM = STAGES * SLOT > OUT ? STAGES * SLOT : OUT;
  static constexpr int OPS = CA + 1 + 4 * TN;  // memory operations of a wave and stage
  static_assert(SI >= 1 && SI < NW && (STAGES - 2) * OPS < 64, "copies per wave");

  floatx16 acc[TN][TM];

  template <typename RowOf, typename Scales>
  __device__ __forceinline__ void run(uint8_t *smem, const uint8_t *a, int64_t a_bytes, const float *as, int64_t as_bytes,
                                      RowOf row_of, int rows, const uint8_t *w, int blocks, const float *ws, int64_t ws_bytes,
                                      Scales ws_of, int k, int KT) {
    const int lane = lane_id(), col = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const rsrc_t ra = make_rsrc(a, a_bytes), rw = make_rsrc(w, (int64_t)min(blocks, BN / 32) * KT * 4096);
    const uint32_t ch = (uint32_t)(((lane & 7) ^ (((wave * 8 + (lane >> 3)) >> 1) & 7)) << 4);
    uint32_t off[CA];
#pragma unroll
    for (int i = 0; i < CA; ++i) {
      const int64_t src = row_of((wave + i * NW) * 8 + (lane >> 3));
      off[i] = src < 0 ? OOB_OFFSET : (uint32_t)(src * k) + ch;
    }
    const bool row_scales = wave < SI;
    const rsrc_t rsc = row_scales ? make_rsrc(as, as_bytes) : make_rsrc(ws, ws_bytes);
    const int sc_at = row_scales ? BM * 128 + wave * 256 : WS_AT;
    uint32_t soff = OOB_OFFSET;
    if (row_scales) {
      const int64_t src = row_of(wave * 64 + lane);
      if (src >= 0) soff = (uint32_t)(src * KT * 4);
    } else if (lane < BN / 32) {
      soff = (uint32_t)(ws_of(lane) * 4);
    }
    intx4 wr[STAGES][TN][4];
    // A stage's copies and loads. Between two barriers, all of them: the waits count them.
    auto issue = [&](auto slot_c, int kt) {
      constexpr int slot = decltype(slot_c)::value;
      uint8_t *sb = smem + slot * SLOT;
      const uint32_t k0 = (uint32_t)kt * 128;
#pragma unroll
      for (int c = 0; c < CA; ++c) bdma16(ra, sb + (wave + c * NW) * 1024, k0 + ch < (uint32_t)k ? off[c] : OOB_OFFSET, k0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsc, LDS_PTR(sb + sc_at), 4, soff, kt * 4, 0, 0);
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          wr[slot][i][q] = __builtin_bit_cast(
              intx4, __builtin_amdgcn_raw_buffer_load_b128(rw, lane * 16, (min(wave * TN + i, blocks - 1) * KT + kt) * 4096 + q * 1024, 0));
    };
    const int swz = (col >> 1) & 7;
    const uint32_t a_off = (uint32_t)(col * 128 + (((2 * h) ^ swz) << 4));
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j) acc[i][j] = floatx16{};
    auto stage = [&](auto slot_c) {
      constexpr int slot = decltype(slot_c)::value;
      const uint8_t *sb = smem + slot * SLOT;
      Fp8Frag<EXACT> wf[TN], x[2];
      float sa[TM], sw[TN];
      auto load_x = [&](int j) {
        const uint8_t *p = sb + j * 32 * 128;
        x[j & 1].set(0, *(const intx4 *)(p + a_off), *(const intx4 *)(p + (a_off ^ 16)));
        x[j & 1].set(1, *(const intx4 *)(p + (a_off ^ 64)), *(const intx4 *)(p + (a_off ^ 80)));
      };
      load_x(0);
#pragma unroll
      for (int j = 0; j < TM; ++j) sa[j] = *(const float *)(sb + BM * 128 + (j * 32 + col) * 4);
#pragma unroll
      for (int i = 0; i < TN; ++i) {
        sw[i] = *(const float *)(sb + WS_AT + (wave * TN + i) * 4);
        wf[i].set(0, wr[slot][i][0], wr[slot][i][1]);
        wf[i].set(1, wr[slot][i][2], wr[slot][i][3]);
      }
      static_for<TM>([&](auto j_c) {
        constexpr int j = decltype(j_c)::value;
        if constexpr (j + 1 < TM) load_x(j + 1);
#pragma unroll
        for (int i = 0; i < TN; ++i) {
          const floatx16 p = fp8_product(wf[i], x[j & 1]);
          const float sc = sa[j] * sw[i];
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][j][r] = __builtin_fmaf(p[r], sc, acc[i][j][r]);
        }
      });
    };
    auto arrived = [&](auto behind_c) {
      __builtin_amdgcn_sched_barrier(0);
      WAIT_VMCNT(decltype(behind_c)::value * OPS);
      WAIT_LGKMCNT0();
      BARRIER();
      __builtin_amdgcn_sched_barrier(0);
    };
    static_for<STAGES - 1>([&](auto d_c) {
      if (decltype(d_c)::value < KT) issue(d_c, decltype(d_c)::value);
    });
    int kt = 0;
    for (; kt + 2 * STAGES - 1 <= KT; kt += STAGES)
      static_for<STAGES>([&](auto d_c) {
        constexpr int d = decltype(d_c)::value;
        arrived(ic<STAGES - 2>{});
        issue(ic<(d + STAGES - 1) % STAGES>{}, kt + d + STAGES - 1);
        stage(d_c);
      });
    for (; kt < KT; kt += STAGES)
      static_for<STAGES>([&](auto d_c) {
        constexpr int d = decltype(d_c)::value;
        if (kt + d < KT) {
          if (kt + d + STAGES - 2 < KT) arrived(ic<STAGES - 2>{});
          else arrived(ic<0>{});
          if (kt + d + STAGES - 1 < KT) issue(ic<(d + STAGES - 1) % STAGES>{}, kt + d + STAGES - 1);
          stage(d_c);
        }
      });
    __syncthreads();
  }
};
