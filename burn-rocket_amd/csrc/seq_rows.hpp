// Attention of sequences with few query rows (decode steps, short chunks) on
// gfx950: the keys of a tile of 16·RT rows are split over the waves of a workgroup
// and, by the plan's items, over workgroups.
//
// Bound by the read of K and V (with few keys by latency): a wave walks the
// item's 32-key chunks on its own (wave w chunks w, w + RW, ...), the next
// chunk's K rows in flight straight to operand registers and its V rows to a
// wave-private LDS buffer (copied as they lie), so that nothing waits on a barrier
// until the softmax states of the waves meet. Per chunk
// (v_mfma_f32_16x16x32):
//   Sᵀ = K·Qᵀ   a lane owns one query row (lane % 16) and keys 4·(lane/16)+e of
//               each 16-key block, so that the row maximum is in the lane and two
//               lane swaps;
//   P           exp2 in f32 against the running maximum, held as two values of the
//               type (the second product costs nothing beside the reads);
//   Oᵀ += Vᵀ·Pᵀ V read back through the transposing LDS read, which hands a lane
//               the keys of P's registers: V needs no rearranging pass.
// A chunk is two 16-key blocks, each inside one page, with a buffer descriptor of
// its own: what lies past the sequence's keys reads as zeros without a branch. The
// addresses of a wave's next 32 chunks wait in registers (lane l: block l).
//
// MI355X: 64 sequences of one token on 100 to 8000 keys, 16/8 heads of 128, 185 us (1.08
// GB, 5.8 TB/s; a copy of 2 GiB moves 4.7); three on 60000 to 131072, 32/4
// heads of 128, 102 us (5.4 TB/s); one token on 4097 keys, 32/4 heads of 128, 10.5
// us: a launch, one trip for the lists, one for K and V, and three for the states.
//
// An item that is one of n_parts of its tile puts its state (Oᵀ unnormalised, m, l)
// into the plan's workspace; the workgroup that arrives last merges all of them in
// key order, whichever it is. Nothing waits on another workgroup.
#pragma once

#include <algorithm>

#include "seq_attn.hpp"

namespace {
constexpr int CK = SEQ_ROWS_CHUNK;  // keys per chunk

template <int D, int RW>
struct SeqRowsGeom {
  static constexpr int NQC = (D + 31) / 32;  // 32-wide d chunks of QKᵀ
  static constexpr int NDB = (D + 15) / 16;  // 16-row d blocks of Oᵀ
  static constexpr int CH = D / 8;           // 16-byte pieces per V row
  static constexpr int VB_INS = (16 * CH + 63) / 64;  // 1 KB copies per 16-key block of V
  static constexpr int VB_BYTES = VB_INS * 1024;
  static constexpr int V_BYTES = 2 * VB_BYTES;
  static constexpr int KL = 2 * NQC;  // K loads per chunk
  static constexpr bool POW2 = (D & (D - 1)) == 0;
  static constexpr int SWZ = POW2 ? (CH / 2 < 8 ? CH / 2 : 8) - 1 : 0;  // swizzle of 32-byte pairs by the key
  static constexpr int SLOT_BYTES = NDB * 1024 + 16 * 8;  // a state: Oᵀ tiles, then (m, l) per row
  static_assert(V_BYTES >= NDB * 1024 && 2 * RW * V_BYTES <= 160 * 1024 && KL + 2 * VB_INS <= 63, "geometry");
};
}  // namespace

// One item for one kv head: `block` counts the kv heads of one item, then the next item.
// v_even, v_odd: the two V buffers of the waves, RW·V_BYTES each and objects of their
// own: the compiler then knows that a copy into one is not what a read of the other
// waits for.
template <int DT, int D, int RW, bool PAGED>
__device__ __forceinline__ void seq_rows_item(const SeqAttnArgs &a, int block, uint8_t *v_even, uint8_t *v_odd) {
  using Gm = SeqRowsGeom<D, RW>;
  constexpr int KBUF = D > 128 ? 1 : 2;  // K register sets (two of head dim 256 spill)
  constexpr int NQC = Gm::NQC, NDB = Gm::NDB, CH = Gm::CH, VB_INS = Gm::VB_INS, KL = Gm::KL;

  const int KV = a.n_kv_heads, G = a.n_head / KV;
  const int kvh = block % KV;
  const SeqItem it = a.rows.items[block / KV];
  if (it.rows == 0) return;
  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, lg = lane >> 4;

  // ---- this lane's row
  const int r = it.row0 + l16;
  const bool rok = r < it.rows;
  const int q = rok ? r / G : 0, h = kvh * G + (rok ? r % G : 0);
  int klo, khi;
  seq_visible(a, it.pos0 + q, it.kv_len, klo, khi);
  if (!rok) khi = -1;
  uintx4 qf[NQC];
  const f16 *qrow = (const f16 *)a.q + (int64_t)(it.tok0 + q) * a.q_stride + (int64_t)h * D;
#pragma unroll
  for (int c = 0; c < NQC; ++c) {
    const int d0 = 32 * c + 8 * lg;
    qf[c] = (rok && d0 < D) ? *(const uintx4 *)(qrow + d0) : uintx4{};
  }
  f16 *const orow = (f16 *)a.out + (int64_t)(it.tok0 + q) * a.out_stride + (int64_t)h * D;
  const bool softcap = a.softcap != 0.f;
  const float C = softcap ? LOG2E : a.scale * LOG2E;

  // ---- K loads and V copies of chunk c (of the sequence)
  const int c_end = (it.k_end + CK - 1) / CK;
  int c = it.k_begin / CK + wave;
  const uint32_t ks = (uint32_t)((PAGED ? D : a.k_stride) * 2), vs = (uint32_t)((PAGED ? D : a.v_stride) * 2);
  const uint32_t k_lane = (uint32_t)l16 * ks + (uint32_t)(lg * 16);
  const int v_wave = wave * Gm::V_BYTES;
  // Blocks of the wave's chunks from win_c on: lane l block l % 2 of the (l / 2)-th.
  KeyBlocks kb{}, vb{};
  int win_c = c;
  auto turn = [&](int from) ALWAYS_INLINE {
    const int key0 = (from + (lane >> 1) * RW) * CK + 16 * (lane & 1);
    const int page = PAGED ? a.table[it.table + (min(key0, it.kv_len - 1) >> a.page_log2)] : 0;
    kb = key_blocks<PAGED>(a, it, a.k, a.k_stride, kvh, key0, page);
    vb = key_blocks<PAGED>(a, it, a.v, a.v_stride, kvh, key0, page);
    win_c = from;
  };
  auto load_k = [&](uintx4(&kf)[2][NQC], int cc) ALWAYS_INLINE {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const rsrc_t rk = block_rsrc(kb, (cc - win_c) / RW * 2 + b);
#pragma unroll
      for (int i = 0; i < NQC; ++i) {
        const uint32_t off = 32 * i + 8 * lg < D ? k_lane + 64 * i : OOB_OFFSET;
        kf[b][i] = __builtin_bit_cast(uintx4, __builtin_amdgcn_raw_buffer_load_b128(rk, off, 0, 0));
      }
    }
  };
  auto copy_v = [&](auto buf_c, int cc) ALWAYS_INLINE {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const rsrc_t rv = block_rsrc(vb, (cc - win_c) / RW * 2 + b);
#pragma unroll
      for (int i = 0; i < VB_INS; ++i) {
        const int p = 64 * i + lane, row = p / CH, ch = p % CH;
        const int lch = Gm::SWZ ? ch ^ ((row & Gm::SWZ) << 1) : ch;  // logical piece of this slot
        uint8_t *const to = (decltype(buf_c)::value ? v_odd : v_even) + (v_wave + b * Gm::VB_BYTES + i * 1024);
        // (row 16 and up, of a ragged last copy, lie past the block's buffer)
        bdma16(rv, to, (uint32_t)row * vs + (uint32_t)(lch * 16), 0);
      }
    }
  };
  // Zeros over the rows of chunk cc that lie below the item's first key.
  auto cut_v = [&](auto buf_c, int cc) ALWAYS_INLINE {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < VB_INS; ++i)
        if (hidden_below(it, cc * CK + 16 * b, (64 * i + lane) / CH))
          *(uintx4 *)((decltype(buf_c)::value ? v_odd : v_even) + (v_wave + b * Gm::VB_BYTES + i * 1024 + lane * 16)) = uintx4{};
  };
  // Transposing reads: this lane's 8 bytes of key 4·lg + l16/4 of a block, columns
  // 16·db + 4·(l16%4)..; the swizzle moves 32-byte pairs.
  const int vkey = 4 * lg + (l16 >> 2);
  const uint32_t v_row = (uint32_t)(vkey * (D * 2) + (l16 & 3) * 8);
  const int vsw = vkey & Gm::SWZ;

  floatx4 o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) o[db] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;
  floatx4 s[2];
  auto scores = [&](const uintx4(&kf)[2][NQC]) ALWAYS_INLINE {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[b] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NQC; ++i) s[b] = mfma16<DT>(kf[b][i], qf[i], s[b]);
    }
  };
  auto softmax_pv = [&](auto buf_c, int cc) ALWAYS_INLINE {
    if (softcap) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[b][e] = a.softcap * tanhf(s[b][e] * a.scale / a.softcap);
    }
    float x[8], mt = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int key = cc * CK + 16 * (i >> 2) + 4 * lg + (i & 3);
      const float sc = a.uniform ? 0.f : s[i >> 2][i & 3] * C;
      x[i] = (key < klo || key > khi) ? -INFINITY : sc;
      mt = fmaxf(mt, x[i]);
    }
    mt = max4groups(mt);
    const float m_new = fmaxf(m_run, mt);
    const float mu = m_new == -INFINITY ? 0.f : m_new;
    if (__builtin_amdgcn_ballot_w64(m_new > m_run) != 0) {
      const float alpha = __builtin_amdgcn_exp2f(m_run - mu);
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < NDB; ++db) o[db] *= alpha;
    }
    m_run = m_new;
    uintx4 p, p_lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e0 = __builtin_amdgcn_exp2f(x[2 * i] - (mu - P_BIAS)), e1 = __builtin_amdgcn_exp2f(x[2 * i + 1] - (mu - P_BIAS));
      l_run += e0 + e1;
      uint32_t hi, lo;
      split2<DT>(e0, e1, hi, lo);
      p[i] = hi;
      p_lo[i] = lo;
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const uint8_t *const at = (decltype(buf_c)::value ? v_odd : v_even) + (v_wave + (int)v_row + ((db ^ vsw) << 5));
      const uintx4 vf = join8(lds_read_tr16(at), lds_read_tr16(at + Gm::VB_BYTES));
      o[db] = mfma16<DT>(vf, p, o[db]);
      o[db] = mfma16<DT>(vf, p_lo, o[db]);
    }
  };

  // ---- the wave's chunks. Loads of a chunk past the last read nothing; with them the
  // loop has one path, on which the number of loads in flight is known.
  uintx4 kf[KBUF][2][NQC];
  auto step = [&](auto cur_c) ALWAYS_INLINE {
    constexpr int CUR = decltype(cur_c)::value;
    const int nx = c + RW;
    if (nx - win_c == 32 * RW) turn(nx);
    if constexpr (KBUF == 2) {
      load_k(kf[CUR ^ 1], nx);
      copy_v(ic<CUR ^ 1>{}, nx);
      asm volatile("" ::: "memory");
      WAIT_VMCNT(KL + 2 * VB_INS);  // this chunk's have landed
      asm volatile("" ::: "memory");
      scores(kf[CUR]);
    } else {  // one K register set: refilled once the scores are formed
      WAIT_VMCNT(0);
      asm volatile("" ::: "memory");
      copy_v(ic<CUR ^ 1>{}, nx);
      scores(kf[0]);
      load_k(kf[0], nx);
    }
    if (c * CK < it.k_lo) cut_v(cur_c, c);
    softmax_pv(cur_c, c);
    WAIT_LGKMCNT0();  // the V buffer's reads are done before it is refilled
    asm volatile("" ::: "memory");
    c = nx;
  };
  if (c < c_end) {
    turn(c);
    load_k(kf[0], c);
    copy_v(ic<0>{}, c);
    while (true) {
      step(ic<0>{});
      if (c >= c_end) break;
      step(ic<1>{});
      if (c >= c_end) break;
    }
    WAIT_VMCNT(0);  // (copies to LDS end before it is used again)
  }

  // ---- the waves' states meet in LDS: (m, l) per row, Oᵀ per lane
  __syncthreads();  // the V buffers are free
  floatx4 *x_o = (floatx4 *)v_even;  // [wave][tile][lane]
  float2 *x_ml = (float2 *)v_odd;    // [wave][16]
  {
    const float l = sum4groups(l_run);
    if (lg == 0) x_ml[wave * 16 + l16] = make_float2(m_run, l);
#pragma unroll
    for (int db = 0; db < NDB; ++db) x_o[(wave * NDB + db) * 64 + lane] = o[db];
  }
  __syncthreads();
  // wave w merges d blocks w, w + RW, ...
  constexpr int SC1 = 16;  // cache policy bit: device scope
  const int S = it.n_parts;
  const uint32_t slot_step = (uint32_t)KV * Gm::SLOT_BYTES;
  const rsrc_t rp = make_rsrc((const uint8_t *)a.rows.part + ((int64_t)it.part0 * KV + kvh) * Gm::SLOT_BYTES,
                              S > 1 ? (int64_t)(S - 1) * slot_step + Gm::SLOT_BYTES : 0);
  const uint32_t mine = (uint32_t)it.sp * slot_step;
  float wa[RW], m_all = -INFINITY, l_all = 0.f;
  {
    float2 ml[RW];
#pragma unroll
    for (int w = 0; w < RW; ++w) {
      ml[w] = x_ml[w * 16 + l16];
      m_all = fmaxf(m_all, ml[w].x);
    }
    const float mu = m_all == -INFINITY ? 0.f : m_all;
#pragma unroll
    for (int w = 0; w < RW; ++w) {
      wa[w] = __builtin_amdgcn_exp2f(ml[w].x - mu);
      l_all += ml[w].y * wa[w];
    }
  }
  auto store_o = [&](int db, floatx4 ov, float inv) ALWAYS_INLINE {
    const int d0 = db * 16 + 4 * lg;
    if (rok && d0 < D) *(uintx2 *)(orow + d0) = uintx2{pack2<DT>(ov[0] * inv, ov[1] * inv), pack2<DT>(ov[2] * inv, ov[3] * inv)};
  };
  for (int db = wave; db < NDB; db += RW) {
    floatx4 ov = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < RW; ++w) ov += x_o[(w * NDB + db) * 64 + lane] * wa[w];
    if (S > 1)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uintx4, ov), rp,
                                             rok ? mine + (uint32_t)((db * 64 + lane) * 16) : OOB_OFFSET, 0, SC1);
    else
      store_o(db, ov, 1.0f / l_all);
  }
  if (S == 1) return;
  if (wave == 0 && lg == 0) {
    const uintx2 w = {__float_as_uint(m_all), __float_as_uint(l_all)};
    __builtin_amdgcn_raw_buffer_store_b64(w, rp, mine + (uint32_t)(NDB * 1024 + l16 * 8), 0, SC1);
  }
  WAIT_VMCNT(0);  // the state is stored before the arrival count
  __syncthreads();
  unsigned *flag = (unsigned *)v_odd;
  if (threadIdx.x == 0) {
    unsigned *cnt = a.rows.cnt + (int64_t)it.part0 * KV + kvh;
    const unsigned last = atomicAdd(cnt, 1u) == (unsigned)(S - 1);
    if (last) atomicExch(cnt, 0u);  // every part is in: reset for the next launch
    *flag = last;
  }
  __syncthreads();
  if (!*flag) return;
  // The parts in key order, MERGE of them in flight together (each load is a trip to memory).
  constexpr int MERGE = 16;
  for (int db = wave; db < NDB; db += RW) {
    float m = -INFINITY, l = 0.f;
    floatx4 ov = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < S; p0 += MERGE) {
      floatx4 x[MERGE];
      uintx2 ml[MERGE];
#pragma unroll
      for (int i = 0; i < MERGE; ++i) {
        const uint32_t slot = rok && p0 + i < S ? (uint32_t)(p0 + i) * slot_step : OOB_OFFSET;  // past the end: zeros
        x[i] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(
                                               rp, slot + (uint32_t)((db * 64 + lane) * 16), 0, SC1));
        ml[i] = __builtin_amdgcn_raw_buffer_load_b64(rp, slot + (uint32_t)(NDB * 1024 + l16 * 8), 0, SC1);
      }
      float mn = m;
#pragma unroll
      for (int i = 0; i < MERGE; ++i) mn = fmaxf(mn, p0 + i < S ? __uint_as_float(ml[i][0]) : -INFINITY);
      const float mu = mn == -INFINITY ? 0.f : mn, al = __builtin_amdgcn_exp2f(m - mu);
      m = mn;
      l *= al;
      ov *= al;
#pragma unroll
      for (int i = 0; i < MERGE; ++i) {
        const float w = p0 + i < S ? __builtin_amdgcn_exp2f(__uint_as_float(ml[i][0]) - mu) : 0.f;
        l += __uint_as_float(ml[i][1]) * w;
        ov += x[i] * w;
      }
    }
    store_o(db, ov, 1.0f / l);
  }
}

template <int DT, int D, int RW, bool PAGED>
__global__ __launch_bounds__(RW * 64, 2) void seq_rows_kernel(SeqAttnArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t v_even[RW * SeqRowsGeom<D, RW>::V_BYTES];
  __shared__ __attribute__((aligned(16))) uint8_t v_odd[RW * SeqRowsGeom<D, RW>::V_BYTES];
  seq_rows_item<DT, D, RW, PAGED>(a, blockIdx.x, v_even, v_odd);
}

namespace {
template <int DT, int D, bool PAGED>
hipError_t launch_seq_rows(const SeqAttnArgs &a, bool brief, hipStream_t st) {
  const dim3 grid((unsigned)(a.rows.n * a.n_kv_heads));
  // Eight waves where their LDS fits; four where no item has more chunks than that
  // half has to itself, as two such workgroups share a CU (24 sequences of 4 to 40
  // tokens, 16/8 heads of 128: 8.2 us against 11.9; 64 sequences of up to 8000 keys the
  // other way round: 197 against 186).
  if constexpr (D <= 128) {
    if (!brief) {
      hipLaunchKernelGGL((seq_rows_kernel<DT, D, 8, PAGED>), grid, dim3(512), 0, st, a);
      return hipGetLastError();
    }
  }
  hipLaunchKernelGGL((seq_rows_kernel<DT, D, 4, PAGED>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

template <int DT, bool PAGED>
hipError_t launch_seq_rows_d(const SeqAttnArgs &a, bool brief, hipStream_t st) {
  switch (a.head_dim) {
    case 32: return launch_seq_rows<DT, 32, PAGED>(a, brief, st);
    case 48: return launch_seq_rows<DT, 48, PAGED>(a, brief, st);
    case 64: return launch_seq_rows<DT, 64, PAGED>(a, brief, st);
    case 72: return launch_seq_rows<DT, 72, PAGED>(a, brief, st);
    case 80: return launch_seq_rows<DT, 80, PAGED>(a, brief, st);
    case 96: return launch_seq_rows<DT, 96, PAGED>(a, brief, st);
    case 112: return launch_seq_rows<DT, 112, PAGED>(a, brief, st);
    case 128: return launch_seq_rows<DT, 128, PAGED>(a, brief, st);
    case 256: return launch_seq_rows<DT, 256, PAGED>(a, brief, st);
  }
  return hipErrorInvalidValue;
}
}  // namespace
