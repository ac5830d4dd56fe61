// Attention of sequences with many query rows (prompts, chunks of prompts) on
// gfx950: an online softmax over key tiles that K and V reach through LDS.
//
// A workgroup's 4 waves have 16·QB query rows of one kv head each (a tile of 128, 64 for
// head dim 256) and walk the item's key tiles of TK keys together: products (P·V of one
// tile, then K·Qᵀ of the next), then the softmax. Two workgroups share a CU, so that
// a SIMD multiplies for a wave of one while it exponentiates for one of the other, and
// so that one's start and end hide behind the other's tiles. One barrier per tile.
//
// Per wave and tile (v_mfma_f32_16x16x32):
//   Sᵀ = K·Qᵀ   K rows from LDS, Q in registers; a lane owns one query of each
//               16-query block and keys 4·(lane/16)+e of each 16-key block;
//   P           exp2 against a maximum that is only raised when a score passes it
//               by 2^RESCALE, held as two values of the type (split2), which takes half
//               as many products again;
//   Oᵀ += Vᵀ·Pᵀ V rows from LDS as they lie in memory, through the transposing
//               read, in the order of P's registers.
// An LDS fragment of K feeds QB products, one of V 2·QB; with 32 rows per wave K's take
// the whole read rate of a CU (128 bytes a clock) while the scores' products run.
//
// Row sums come from the same products (a row of ones), which takes their additions
// off the softmax slot and counts the probabilities as they are held.
//
// LDS: K rows of KPC 16-byte pieces (piece c of row r at c ^ (r & (KPC-1))), V as
// 16-key blocks (32-byte pairs swizzled by the key where rows are a power of two).
// Two buffers of each. Copies go to LDS directly, one 16-key block per buffer
// descriptor: a block lies in one page, and rows past the sequence's keys read as
// zeros. They start with the softmax, which their latency hides behind; issued between
// products they held those up.
//
// MI355X: two prompts of 7000 tokens, 32/4 heads of 128, causal, bf16, 996 us: 0.83 PFLOP/s,
// with the second half of P and the row sums 1.35 issued (the library's 8192³ product reaches
// 1.2). With P as one value it took 742. 512 rows of 8 heads on 16901 keys 187 us (one value:
// 147). 64 passages of 100 to 512 tokens 88 us (79): items of three key
// tiles, whose first loads and last stores nothing hides. Head dim 256 has one 16-query
// block per wave: every score's product reads its own 1 KB from LDS, twice the CU's rate. 49 to 58 us
// for 9261 tokens, 3/1 heads, 512 keys to either side (one value of P: 44 to 52; 128 rows a workgroup,
// one per CU, a quarter more).
//
// Times beside the code that compare two forms were taken with P as one value.
//
// Items that are one of n_parts of their tile leave their state in the plan's
// workspace; the last to arrive merges the parts in key order.
#pragma once

#include "seq_rows.hpp"

namespace {
// LDS fragments read ahead of their products: 2 and 4 to 8 and 8 measured alike.
constexpr int AHEAD_V = 3, AHEAD_K = 4;
constexpr float RESCALE = 8.0f;  // with P_BIAS: probabilities stay below 2^14

template <int D>
struct SeqTilesGeom {
  static constexpr int QB = D <= 128 ? 2 : 1;       // 16-query blocks per wave
  static constexpr int TK = D <= 128 ? 64 : 32;     // keys per tile
  static constexpr int ROWS = 64 * QB;              // query rows per workgroup
  static constexpr int NQC = (D + 31) / 32;         // 32-wide d chunks of QKᵀ
  static constexpr int NDB = (D + 15) / 16;         // 16-row d blocks of Oᵀ
  static constexpr int CH = D / 8;                  // 16-byte pieces of a row
  static constexpr int KPC = D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32;  // pieces per K row in LDS
  static constexpr int KSW = (KPC < 16 ? KPC : 16) - 1;
  static constexpr int KROW = 16 * KPC;
  static constexpr int NB = TK / 16;                // 16-key blocks per tile
  static constexpr int NC2 = TK / 32;               // 32-key chunks per tile
  static constexpr int KI = 16 * KPC / 64;          // 1 KB copies per block of K
  static constexpr int VI = (16 * CH + 63) / 64;    // and of V
  static constexpr int VB = VI * 1024;              // bytes of a V block
  static constexpr bool POW2 = (D & (D - 1)) == 0;
  static constexpr int VSW = POW2 ? (CH / 2 < 8 ? CH / 2 : 8) - 1 : 0;
  static constexpr int K_BYTES = TK * KROW, V_BYTES = NB * VB;
  static constexpr bool WITH_ROWS = seq_one_launch(D);
  static constexpr int ROW_BYTES = WITH_ROWS ? 4 * SeqRowsGeom<D, 4>::V_BYTES : 0;
  static constexpr int K_SMEM = 2 * K_BYTES > ROW_BYTES ? 2 * K_BYTES : ROW_BYTES;
  static constexpr int V_SMEM = 2 * V_BYTES > ROW_BYTES ? 2 * V_BYTES : ROW_BYTES;
  static constexpr int CK = KI * NB / 4, CV = VI * NB / 4;  // copies per wave and tile
  static_assert(KI * NB % 4 == 0 && VI * NB % 4 == 0, "every wave copies alike");
  static constexpr int NJ = 1 + NDB * QB;           // 1 KB pieces of a wave's state in the workspace
  static constexpr int SLOT_BYTES = 4 * NJ * 1024;
  static_assert(2 * (K_SMEM + V_SMEM) <= 160 * 1024, "two workgroups per CU");
};
}  // namespace

// One item for one kv head, with the buffers of K and V.
template <int DT, int D, bool PAGED, bool SOFTCAP>
__device__ __forceinline__ void seq_tiles_item(const SeqAttnArgs &a, int block, uint8_t *k_smem, uint8_t *v_smem) {
  using Gm = SeqTilesGeom<D>;
  constexpr int QB = Gm::QB, TK = Gm::TK, NQC = Gm::NQC, NDB = Gm::NDB, NB = Gm::NB, NC2 = Gm::NC2;
  constexpr int KI = Gm::KI, VI = Gm::VI, CH = Gm::CH, KPC = Gm::KPC, KROW = Gm::KROW;

  const int KV = a.n_kv_heads, G = a.n_head / KV;
  const int kvh = block % KV;
  const SeqItem it = a.tiles.items[block / KV];
  if (it.rows == 0) return;
  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, lg = lane >> 4;

  // ---- this lane's rows and what they see. A negative scale is a sign of Q.
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
  const float scale = fabsf(a.scale);
  bool rok[QB];
  int klo[QB], khi[QB];
  uintx4 qf[QB][NQC];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int r = it.row0 + wave * 16 * QB + qb * 16 + l16;
    rok[qb] = r < it.rows;
    const int q = rok[qb] ? r / G : 0, h = kvh * G + (rok[qb] ? r % G : 0);
    seq_visible(a, it.pos0 + q, it.kv_len, klo[qb], khi[qb]);
    if (!rok[qb]) khi[qb] = -1;
    const f16 *qrow = (const f16 *)a.q + (int64_t)(it.tok0 + q) * a.q_stride + (int64_t)h * D;
#pragma unroll
    for (int c = 0; c < NQC; ++c) {
      const int d0 = 32 * c + 8 * lg;
      qf[qb][c] = ((rok[qb] && d0 < D) ? *(const uintx4 *)(qrow + d0) : uintx4{}) ^ flip;
    }
  }
  // Keys that every row of the wave sees, from its first and last row (the ends of
  // a row's keys never decrease with the row).
  int full_lo, full_hi, skip;
  const int w_row0 = min(it.row0 + wave * 16 * QB, it.rows - 1);
  seq_visible(a, it.pos0 + w_row0 / G, it.kv_len, skip, full_hi);
  seq_visible(a, it.pos0 + min(w_row0 + 16 * QB - 1, it.rows - 1) / G, it.kv_len, full_lo, skip);
  // (a scale of 0 must leave hidden scores at -inf)
  const float C = SOFTCAP ? LOG2E : scale != 0.f ? scale * LOG2E : 1e-30f;

  // ---- copies
  const uint32_t ks = (uint32_t)((PAGED ? D : a.k_stride) * 2), vs = (uint32_t)((PAGED ? D : a.v_stride) * 2);
  // Tiles kt_begin + j, the first with the first key that a row sees.
  const int kt_begin = max(it.k_begin, it.k_lo) / TK, nj = (it.k_end + TK - 1) / TK - kt_begin;
  // Blocks of the item's tiles: lane l holds block l % NB of tile l / NB of a window
  // of WIN tiles; kb and vb: of the windows that the next copies of K and V lie in;
  // ids: page ids of the window that comes next (fetched a window ahead).
  constexpr int WIN = 64 / NB;
  KeyBlocks kb, vb;
  int ids = 0;
  auto key_of = [&](int w) ALWAYS_INLINE { return (kt_begin + w * WIN + lane / NB) * TK + 16 * (lane % NB); };
  auto fetch_ids = [&](int w) ALWAYS_INLINE {
    if constexpr (PAGED) ids = a.table[it.table + (min(key_of(w), it.kv_len - 1) >> a.page_log2)];
  };
  auto turn_k = [&](int w) ALWAYS_INLINE { kb = key_blocks<PAGED>(a, it, a.k, a.k_stride, kvh, key_of(w), ids); };
  auto turn_v = [&](int w) ALWAYS_INLINE { vb = key_blocks<PAGED>(a, it, a.v, a.v_stride, kvh, key_of(w), ids); };
  // The wave's share of the copies of tile j: pieces s of its 16-key
  // blocks b, in the order s + KI·b.
  auto k_buf = [&](int j) ALWAYS_INLINE { return k_smem + (j & 1) * Gm::K_BYTES; };
  auto v_buf = [&](int j) ALWAYS_INLINE { return v_smem + (j & 1) * Gm::V_BYTES; };
  auto copy_k = [&](int j) ALWAYS_INLINE {
    uint8_t *const to = k_buf(j);
    static_for<Gm::CK>([&](auto i_c) ALWAYS_INLINE {
      const int c = wave + 4 * decltype(i_c)::value, b = c / KI, s = c % KI;
      const rsrc_t rk = block_rsrc(kb, (j % WIN) * NB + b);
      const int p = 64 * s + lane, row = p / KPC;
      const int ch = (p % KPC) ^ (row & Gm::KSW);  // logical piece of this slot
      bdma16(rk, to + c * 1024, ch < CH ? (uint32_t)row * ks + (uint32_t)(ch * 16) : OOB_OFFSET, 0);
    });
  };
  auto copy_v = [&](int j) ALWAYS_INLINE {
    uint8_t *const to = v_buf(j);
    static_for<Gm::CV>([&](auto i_c) ALWAYS_INLINE {
      const int c = wave + 4 * decltype(i_c)::value, b = c / VI, s = c % VI;
      const rsrc_t rv = block_rsrc(vb, (j % WIN) * NB + b);
      const int p = 64 * s + lane, row = p / CH, ch = p % CH;
      const int lch = Gm::VSW ? ch ^ ((row & Gm::VSW) << 1) : ch;
      // (row 16 and up, of a ragged last copy, lie past the block's buffer)
      bdma16(rv, to + c * 1024, (uint32_t)row * vs + (uint32_t)(lch * 16), 0);
    });
  };

  // Zeros over the rows of the wave's own copies of the first tile that lie below that key
  // (with a comparison in every copy two long prompts took 760 us instead of 742).
  auto cut_v = [&] ALWAYS_INLINE {
    static_for<Gm::CV>([&](auto i_c) ALWAYS_INLINE {
      const int c = wave + 4 * decltype(i_c)::value, b = c / VI, s = c % VI;
      if (hidden_below(it, kt_begin * TK + 16 * b, (64 * s + lane) / CH))
        *(uintx4 *)(v_smem + c * 1024 + lane * 16) = uintx4{};
    });
    WAIT_LGKMCNT0();
  };

  // ---- LDS fragment addresses
  uint32_t k_off[NQC];
#pragma unroll
  for (int c = 0; c < NQC; ++c) k_off[c] = (uint32_t)(l16 * KROW + (((4 * c + lg) ^ (l16 & Gm::KSW)) << 4));
  const int vkey = 4 * lg + (l16 >> 2);
  const uint32_t v_row = (uint32_t)(vkey * (D * 2) + (l16 & 3) * 8);
  const int vsw = vkey & Gm::VSW;

  floatx4 o[NDB][QB], s[NB][QB];
  uintx4 p[NC2][QB], p_lo[NC2][QB];
  float m_run[QB];
  floatx4 l_run[QB];  // (every row of the product with ones is the row sum)
  const uint32_t one2 = DT == RK_DTYPE_F16 ? 0x3c003c00u : 0x3f803f80u;
  const uintx4 ones = {one2, one2, one2, one2};
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    m_run[qb] = -INFINITY;
    l_run[qb] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int db = 0; db < NDB; ++db) o[db][qb] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  auto products = [&](int j) ALWAYS_INLINE {
    __builtin_amdgcn_s_setprio(1);  // products first: what they leave of the issue slots is enough for a softmax
    if (j >= 1 && j - 1 < nj) {
      const uint8_t *vt = v_buf(j - 1) + v_row;
#pragma unroll
      for (int c2 = 0; c2 < NC2; ++c2) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          l_run[qb] = mfma16<DT>(ones, p[c2][qb], l_run[qb]);
          l_run[qb] = mfma16<DT>(ones, p_lo[c2][qb], l_run[qb]);
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const uint8_t *at = vt + 2 * c2 * Gm::VB + ((db ^ vsw) << 5);
          const uintx4 vf = join8(lds_read_tr16(at), lds_read_tr16(at + Gm::VB));
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) o[db][qb] = mfma16<DT>(vf, p[c2][qb], o[db][qb]);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) o[db][qb] = mfma16<DT>(vf, p_lo[c2][qb], o[db][qb]);
        }
      }
      // Each fragment (two reads) AHEAD_V fragments ahead of its products.
      constexpr int NF = NC2 * NDB, AV = AHEAD_V < NF ? AHEAD_V : NF;
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * AV, 0);
      static_for<NF - AV>([&](auto) ALWAYS_INLINE {
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * QB, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      });
      __builtin_amdgcn_sched_group_barrier(0x008, 2 * QB * (AV + NC2), 0);
    }
    __builtin_amdgcn_sched_barrier(0);  // P dies before S is made
    if (j < nj) {
      const uint8_t *kt = k_buf(j);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) s[b][qb] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NQC; ++c)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uintx4 kf = *(const uintx4 *)(kt + k_off[c] + b * 16 * KROW);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) s[b][qb] = mfma16<DT>(kf, qf[qb][c], s[b][qb]);
        }
      constexpr int NR = NB * NQC, AK = AHEAD_K < NR ? AHEAD_K : NR;
      __builtin_amdgcn_sched_group_barrier(0x100, AK, 1);
      static_for<NR - AK>([&](auto) ALWAYS_INLINE {
        __builtin_amdgcn_sched_group_barrier(0x008, QB, 1);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
      });
      __builtin_amdgcn_sched_group_barrier(0x008, QB * AK, 1);
    }
  };
  auto softmax = [&](int j) ALWAYS_INLINE {
    __builtin_amdgcn_s_setprio(0);
    // The copies (past the last tile of zeros; page ids land with them). Their buffers
    // were last read before the barrier that every wave has passed.
    if ((j + 1) % WIN == 0) turn_k(j / WIN + 1);
    if (j % WIN == 0) turn_v(j / WIN);
    copy_k(j + 1);
    copy_v(j);
    if (j % WIN == 0) fetch_ids(j / WIN + 1);
    const int key0 = (kt_begin + j) * TK;
    if constexpr (SOFTCAP) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[b][qb][e] = a.softcap * tanhf(s[b][qb][e] * scale / a.softcap);
    }
    const auto each = [&](auto f) ALWAYS_INLINE {  // (s, its key from the lane's first of the tile on, query block)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[b][qb][e] = f(s[b][qb][e], 16 * b + e, qb);
    };
    // One comparison an element, and only on the tiles that an end of the keys crosses: both
    // ends and `uniform` tested at once took 80.4 us for the passages, 79.4 so, and 145 to 143
    // for the 512 rows.
    const int lane_key = key0 + 4 * lg;
    if (a.uniform) each([](float, int, int) ALWAYS_INLINE { return 0.f; });
    if (key0 + TK - 1 > full_hi)
      each([&](float x, int k, int qb) ALWAYS_INLINE { return k > khi[qb] - lane_key ? -INFINITY : x; });
    if (key0 < full_lo)
      each([&](float x, int k, int qb) ALWAYS_INLINE { return k < klo[qb] - lane_key ? -INFINITY : x; });
    float mt[QB];
    bool up = false;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      float m = s[0][qb][0];
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (b | e) m = __builtin_elementwise_maximum(m, s[b][qb][e]);  // (v_maximum3; fmaxf canonicalizes first)
      mt[qb] = max4groups(m) * C;
      up |= mt[qb] > m_run[qb] + RESCALE;
    }
    if (__builtin_amdgcn_ballot_w64(up) != 0) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const float m_new = fmaxf(m_run[qb], mt[qb]);
        const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run[qb] - m_new);
        m_run[qb] = m_new;
        l_run[qb] *= alpha;
#pragma unroll
        for (int db = 0; db < NDB; ++db) o[db][qb] *= alpha;
      }
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const float nm = m_run[qb] == -INFINITY ? 0.f : P_BIAS - m_run[qb];
#pragma unroll
      for (int c2 = 0; c2 < NC2; ++c2)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int b = 2 * c2 + (i >> 1), e = 2 * (i & 1);
          const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][qb][e], C, nm));
          const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][qb][e + 1], C, nm));
          uint32_t hi, lo;
          split2<DT>(e0, e1, hi, lo);
          p[c2][qb][i] = hi;
          p_lo[c2][qb][i] = lo;
        }
    }
    // P is made here: left alone, the compiler moves the exponentials to their use, into
    // the products.
#pragma unroll
    for (int c2 = 0; c2 < NC2; ++c2)
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) asm volatile("" : "+v"(p[c2][qb]), "+v"(p_lo[c2][qb]));
    __builtin_amdgcn_sched_barrier(0);
    WAIT_VMCNT(0);
  };

  fetch_ids(0);
  turn_k(0);
  copy_k(0);
  WAIT_VMCNT(0);
  BARRIER();
  products(0);
  softmax(0);
  if (kt_begin * TK < it.k_lo) cut_v();
  BARRIER();
  for (int j = 1; j < nj; ++j) {
    products(j);
    softmax(j);
    BARRIER();
  }
  products(nj);
  WAIT_VMCNT(0);
  float l_all[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) l_all[qb] = l_run[qb][0];
  // The wave's rows go out through its quarter of the K buffers (which no wave reads any
  // more), so that a store writes whole rows, 16 bytes a lane: 64 passages of 100 to 512
  // tokens, 16/8 heads of 128, took 85 us with the lanes' own 8 bytes stored from
  // registers (32 bytes a row and store), 81 so.
  auto store_rows = [&](const floatx4(&x)[NDB][QB], const float(&l)[QB]) ALWAYS_INLINE {
    uint8_t *const mine = k_smem + wave * 16 * QB * KROW;
    // (where the rows go is made here: kept over the loop it costs head dim 64 the registers
    // of its third wave a SIMD, and the mixed step 25.8 us instead of 23.3)
    int ln = lane;
    asm volatile("" : "+v"(ln));
    f16 *orow[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int r = it.row0 + wave * 16 * QB + qb * 16 + (ln & 15);
      orow[qb] = r < it.rows ? (f16 *)a.out + (int64_t)(it.tok0 + r / G) * a.out_stride + (int64_t)(kvh * G + r % G) * D : nullptr;
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const float inv = 1.0f / l[qb];
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const int c = 2 * db + (lg >> 1);  // 16-byte piece of row 16·qb + l16
        *(uintx2 *)(mine + (16 * qb + l16) * KROW + ((c ^ (l16 & Gm::KSW)) << 4) + (lg & 1) * 8) =
            uintx2{pack2<DT>(x[db][qb][0] * inv, x[db][qb][1] * inv), pack2<DT>(x[db][qb][2] * inv, x[db][qb][3] * inv)};
      }
    }
    WAIT_LGKMCNT0();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < (16 * QB * CH + 63) / 64; ++i) {
      const int p = 64 * i + lane, row = p / CH, ch = p % CH;
      uint64_t at[QB];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
        at[qb] = (uint64_t)__shfl((unsigned)((uint64_t)orow[qb] >> 32), row & 15, 64) << 32 |
                 (uint32_t)__shfl((unsigned)(uint64_t)orow[qb], row & 15, 64);
      uint8_t *const to = (uint8_t *)(QB == 1 || row < 16 ? at[0] : at[QB - 1]);
      if (row < 16 * QB && to)
        *(uintx4 *)(to + ch * 16) = *(const uintx4 *)(mine + row * KROW + ((ch ^ (row & Gm::KSW)) << 4));
    }
  };
  const int S = it.n_parts;
  if (S == 1) {
    store_rows(o, l_all);
    return;
  }
  // ---- one of several parts: the state to its slot, with device-coherent (sc1)
  // accesses; slot: [wave][piece][lane] 16 bytes, piece 0 the (m, l) pairs, piece
  // 1 + db·QB + qb the Oᵀ block.
  constexpr int SC1 = 16;
  constexpr int NJ = Gm::NJ;
  const uint32_t slot_step = (uint32_t)KV * Gm::SLOT_BYTES;
  const rsrc_t rp = make_rsrc((const uint8_t *)a.tiles.part + ((int64_t)it.part0 * KV + kvh) * Gm::SLOT_BYTES,
                              (int64_t)(S - 1) * slot_step + Gm::SLOT_BYTES);
  const uint32_t lane_at = (uint32_t)((wave * NJ * 64 + lane) * 16);
  const uint32_t to = lane_at + (uint32_t)it.sp * slot_step;
  const floatx4 ml_all = {m_run[0], l_all[0], m_run[QB - 1], l_all[QB - 1]};
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uintx4, ml_all), rp, to, 0, SC1);
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uintx4, o[db][qb]), rp,
                                             to + (uint32_t)((1 + db * QB + qb) * 1024), 0, SC1);
  WAIT_VMCNT(0);  // stored before the arrival count
  BARRIER();  // (the K and V buffers are free)
  unsigned *flag = (unsigned *)v_smem;  // (the rows go out through the K buffers)
  if (threadIdx.x == 0) {
    unsigned *cnt = a.tiles.cnt + (int64_t)it.part0 * KV + kvh;
    const unsigned last = atomicAdd(cnt, 1u) == (unsigned)(S - 1);
    if (last) atomicExch(cnt, 0u);  // every part is in: reset for the next launch
    *flag = last;
    WAIT_LGKMCNT0();
  }
  BARRIER();
  if (!*flag) return;
  // The parts in key order.
  float m[QB], l[QB];
  floatx4 acc[NDB][QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    m[qb] = -INFINITY;
    l[qb] = 0.f;
#pragma unroll
    for (int db = 0; db < NDB; ++db) acc[db][qb] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  for (int sp = 0; sp < S; ++sp) {
    const uint32_t at = lane_at + (uint32_t)sp * slot_step;
    const floatx4 ml = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(rp, at, 0, SC1));
    floatx4 x[NDB][QB];
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
        x[db][qb] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(
                                                    rp, at + (uint32_t)((1 + db * QB + qb) * 1024), 0, SC1));
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const float m1 = qb ? ml[2] : ml[0], l1 = qb ? ml[3] : ml[1];
      const float mn = fmaxf(m[qb], m1), mu = mn == -INFINITY ? 0.f : mn;
      const float a0 = __builtin_amdgcn_exp2f(m[qb] - mu), a1 = __builtin_amdgcn_exp2f(m1 - mu);
      m[qb] = mn;
      l[qb] = l[qb] * a0 + l1 * a1;
#pragma unroll
      for (int db = 0; db < NDB; ++db) acc[db][qb] = acc[db][qb] * a0 + x[db][qb] * a1;
    }
  }
  store_rows(acc, l);
}

// The tile items, then the batch's row items: those are bound by their reads of the
// cache and run beside the products of the tiles, or where tiles have ended. MI355X, a
// launch for each list against this one: 24 tokens on up to 2000 keys with a prompt
// chunk of 256 on 2000, 16/4 heads of 64, 25.5 us, 16.8; 64 on up to 8000 with two
// chunks of 1000, 32/4 heads of 128, 206, 147. Row items first: 20.1 and 161; both in
// turns: 18.8 and 145. The most that it lost (64 on up to 8000 with a chunk of 512 on
// 16901, 16/8 heads of 128; row items have half the waves here): 260, 270.
template <int DT, int D, bool PAGED, bool SOFTCAP>
__global__ __launch_bounds__(256, 2) void seq_tiles_kernel(SeqAttnArgs a) {
  using Gm = SeqTilesGeom<D>;
  __shared__ __attribute__((aligned(16))) uint8_t k_smem[Gm::K_SMEM];
  __shared__ __attribute__((aligned(16))) uint8_t v_smem[Gm::V_SMEM];
  const int n_tiles = a.tiles.n * a.n_kv_heads;
  if constexpr (Gm::WITH_ROWS) {
    if ((int)blockIdx.x >= n_tiles) {
      seq_rows_item<DT, D, 4, PAGED>(a, blockIdx.x - n_tiles, k_smem, v_smem);
      return;
    }
  }
  seq_tiles_item<DT, D, PAGED, SOFTCAP>(a, blockIdx.x, k_smem, v_smem);
}

namespace {
template <int DT, int D, bool PAGED, bool SOFTCAP>
hipError_t launch_seq_tiles(const SeqAttnArgs &a, hipStream_t st) {
  using Gm = SeqTilesGeom<D>;
  static_assert(Gm::ROWS == seq_tile_rows(D) && SEQ_KEY_TILE % Gm::TK == 0, "the plan's tiles");
  const dim3 grid((unsigned)((a.tiles.n + a.rows.n) * a.n_kv_heads));
  hipLaunchKernelGGL((seq_tiles_kernel<DT, D, PAGED, SOFTCAP>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

template <int DT, bool PAGED, bool SOFTCAP>
hipError_t launch_seq_tiles_d(const SeqAttnArgs &a, hipStream_t st) {
  switch (a.head_dim) {
    case 32: return launch_seq_tiles<DT, 32, PAGED, SOFTCAP>(a, st);
    case 48: return launch_seq_tiles<DT, 48, PAGED, SOFTCAP>(a, st);
    case 64: return launch_seq_tiles<DT, 64, PAGED, SOFTCAP>(a, st);
    case 72: return launch_seq_tiles<DT, 72, PAGED, SOFTCAP>(a, st);
    case 80: return launch_seq_tiles<DT, 80, PAGED, SOFTCAP>(a, st);
    case 96: return launch_seq_tiles<DT, 96, PAGED, SOFTCAP>(a, st);
    case 112: return launch_seq_tiles<DT, 112, PAGED, SOFTCAP>(a, st);
    case 128: return launch_seq_tiles<DT, 128, PAGED, SOFTCAP>(a, st);
    case 256: return launch_seq_tiles<DT, 256, PAGED, SOFTCAP>(a, st);
  }
  return hipErrorInvalidValue;
}
}  // namespace
