// Products of few rows with a block-scaled fp8 weight: decode steps of a dense layer, and expert tiles of at most 32 rows.
//
// These are bound by the weight's bytes and, below a few MB, by latency: no wave may wait for another while it streams. A
// workgroup's eight waves are `groups` groups that take a 32-row block of the weight each (of an expert's first product: a
// gate and its up block) and split its K among their waves: 4 KB blocks in four 1 KB pieces, straight into the registers
// that a 32 × 32 product reads them from, the next ones on the way. The partial sums meet in LDS, in wave order. (Workgroups
// that do several blocks one behind the other, asking for the next one's weights before they sum up the last, gain 2 % on 64
// tokens of a 30B-A3B layer, and lose more on one.)
//
// The rows (32 columns of the products, most of them empty in a decode step) come as x itself: the workgroup quantizes them
// into LDS once, while its first weights are on the way, so that a layer is one launch; or, where they are more, as codes
// that each wave reads from the caches, whole lines at a time, one or two column blocks a wave.
//
// MI355X: a row through 5120 × 2048 4.3 us (2.4 TB/s), through 16384 × 2048 8.0 (4.2); the experts' products of 64 tokens of that
// layer 76 and 37 us (5.2 and 5.3 TB/s); codes of 48 rows through 2048 × 4096 6.9, of 333 through 1000 × 1104 in f32 6.0.
#include "fp8.hpp"
#include "kernels.hpp"

namespace {
enum { FEW_DENSE = 0, FEW_GATE_UP = 1, FEW_DOWN = 2 };
constexpr int FNW = 8;  // waves, the split of K
constexpr int FEW_CODES = 3;  // x's type: codes and scales

// Bytes of a quantized row in LDS: 16 more than its codes, which spreads the rows over the banks.
__host__ __device__ constexpr int few_row(int kt) { return kt * 128 + 16; }
// Columns of the sums in LDS: a multiple of 8.
__host__ __device__ constexpr int few_cols(int rows) { return rows >= 32 ? 32 : (rows + 7) / 8 * 8; }
// Quantized rows with their scales, and the waves' sums behind them; or codes on their way to the operands, a part of K per
// wave, where the sums go afterwards.
__host__ __device__ constexpr size_t few_in(int rows, int kt) { return ((size_t)rows * (few_row(kt) + kt * 4) + 15) / 16 * 16; }
__host__ __device__ constexpr size_t few_smem(int xt, int nout, int tm, int rows, int kt) {
  const size_t red = (size_t)FNW * nout * 128 * few_cols(rows);
  return xt != FEW_CODES ? few_in(rows, kt) + red : red > (size_t)FNW * tm * 4096 ? red : (size_t)FNW * tm * 4096;
}

// Rows of x to codes in LDS, [row][few_row], by the whole workgroup: 16 lanes a block. Their scales [row][kt] are behind them.
__device__ __forceinline__ float *few_scales(uint8_t *smem, int rows, int kt) { return (float *)(smem + (size_t)rows * few_row(kt)); }
// Block b of the rows: the lane's eight values.
template <int XT, typename RowOf>
__device__ __forceinline__ void few_load(dt_raw<XT, 8> &raw, const void *x, int b, int rows, int k, int kt, RowOf row_of) {
  const int r = b / kt, c = (b - r * kt) * 128 + (threadIdx.x & 15) * 8;
#pragma unroll
  for (int e = 0; e < raw.WORDS; ++e) raw.w[e] = 0;
  if (r >= rows || c >= k) return;
  const int64_t at = row_of(r) * k + c;
  if constexpr (XT == RK_DTYPE_F32) {
    *(uintx4 *)raw.w = *(const uintx4 *)((const float *)x + at);
    *(uintx4 *)(raw.w + 4) = *(const uintx4 *)((const float *)x + at + 4);
  } else {
    *(uintx4 *)raw.w = *(const uintx4 *)((const uint16_t *)x + at);
  }
}
// raw: the thread's first block, loaded by the caller (in front of the weights: what is asked for first comes first).
template <int XT, int NW = FNW, typename RowOf>
__device__ __forceinline__ void few_quantize(uint8_t *smem, dt_raw<XT, 8> &raw, const void *x, int rows, int k, int kt, RowOf row_of) {
  float *s_as = few_scales(smem, rows, kt);
  const int sub = threadIdx.x & 15;
  for (int b = threadIdx.x / 16; b < rows * kt; b += NW * 4) {
    const int r = b / kt, at = b - r * kt;
    float v[8], amax = 0.f;
    dt_decode_raw<XT, 8>(raw, v);
    if (b + NW * 4 < rows * kt) few_load<XT>(raw, x, b + NW * 4, rows, k, kt, row_of);
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(v[e]));
    const float s = fp8_scale(fp8_max16(amax));
    const Fp8Div div(s);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = div(v[e]);
    *(uintx2 *)(smem + (size_t)r * few_row(kt) + at * 128 + sub * 8) =
        uintx2{fp8_codes4(v[0], v[1], v[2], v[3]), fp8_codes4(v[4], v[5], v[6], v[7])};
    if (sub == 0) s_as[r * kt + at] = s;
  }
}
}  // namespace

template <int XT, int MODE, bool EXACT, int TM>
__global__ __launch_bounds__(FNW * 64, 2) void fp8_few_kernel(const Fp8FewArgs g) {
  constexpr int NB = MODE == FEW_GATE_UP ? 2 : 1;  // weight blocks
  constexpr int D = XT == FEW_CODES ? 4 / TM : NB == 2 ? 2 : 4;  // blocks of K on the way, per wave
  static_assert(XT == FEW_CODES || TM == 1, "x in LDS: one column block");
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int lane = lane_id(), col = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kt = g.kt, groups = g.groups, kw = FNW / groups;
  const int grp = wave / kw, wk = wave - grp * kw;  // the wave's group, and its part of K
  // (a tile's workgroups one behind the other: they share its rows)
  const int n_nb = (g.n + 31) / 32, per = (n_nb + groups - 1) / groups, nb0 = blockIdx.x % per * groups;
  const int nb = min(nb0 + grp, n_nb - 1);  // (groups past the last block repeat it: they are not stored)
  int rows = g.m;
  int64_t row0 = 0;
  const uint8_t *w = g.w;
  const float *ws = g.ws;
  if constexpr (MODE != FEW_DENSE) {
    const MoeTile tile = g.tiles[blockIdx.x / per];
    if (tile.rows <= 0 || tile.expert < 0) return;
    rows = tile.rows;
    row0 = tile.row0;
    w += (int64_t)tile.expert * g.w_stride;
    ws += (int64_t)tile.expert * g.ws_stride;
  } else {
    row0 = (int64_t)(blockIdx.x / per) * 32 * TM;
    rows = min((int)(g.m - row0), 32 * TM);
  }

  // Columns past the last row repeat it: they are not stored.
  int row[TM];
#pragma unroll
  for (int j = 0; j < TM; ++j) row[j] = min(j * 32 + col, rows - 1);
  // The wave's parts wk, wk + kw, .. of K, part `it` of them in registers it mod D. Weight blocks of a pair are consecutive
  // in the layout; scales: of the gate rows, then of the up rows.
  const int n_it = (kt - wk + kw - 1) / kw;  // (may be 0)
  const uint8_t *wb = w + ((int64_t)nb * NB * kt + wk) * 4096 + lane * 16;
  const float *wsb = ws + (int64_t)(nb / 4) * kt;
  struct Part {
    intx4 w[NB][4], x[XT == FEW_CODES ? TM : 1][4];
    float sw[NB], sa[TM];
  } ring[D];
  auto load = [&](auto d_c, int it) {
    Part &r = ring[decltype(d_c)::value];
    const int t = wk + kw * it;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[b][i] = *(const intx4 *)(wb + ((int64_t)b * kt + kw * it) * 4096 + i * 1024);
      r.sw[b] = wsb[(int64_t)b * g.up_scales + t];
    }
    if constexpr (XT == FEW_CODES) {
      // whole lines: eight lanes a row of 128 codes
      const int at = t * 128 + (lane & 7) * 16;
#pragma unroll
      for (int j = 0; j < TM; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t src = row0 + min(j * 32 + i * 8 + (lane >> 3), rows - 1);
          r.x[j][i] = at < g.k ? *(const intx4 *)((const uint8_t *)g.x + src * g.k + at) : intx4{0, 0, 0, 0};
        }
        r.sa[j] = g.as[(row0 + row[j]) * kt + t];
      }
    }
  };
  // The first rows of x in front of the weights, unless their addresses come from memory too.
  const auto row_of = [&](int r) -> int64_t {
    if constexpr (MODE == FEW_GATE_UP) return g.top_k > 0 ? (row0 + r) / g.top_k : (int64_t)min(g.tok[row0 + r], g.n_tok - 1);
    return row0 + r;
  };
  constexpr int XQ = XT == FEW_CODES ? RK_DTYPE_F16 : XT;
  dt_raw<XQ, 8> raw;
  const bool early = MODE != FEW_GATE_UP || g.top_k > 0;
  if constexpr (XT != FEW_CODES) {
    if (early) few_load<XQ>(raw, g.x, threadIdx.x / 16, rows, g.k, kt, row_of);
    __builtin_amdgcn_sched_barrier(0);
  }
  static_for<D>([&](auto d_c) {
    if (decltype(d_c)::value < n_it) load(d_c, decltype(d_c)::value);
  });

  const float *s_as = few_scales(smem, rows, kt);
  if constexpr (XT != FEW_CODES) {
    __builtin_amdgcn_sched_barrier(0);
    if (!early) few_load<XQ>(raw, g.x, threadIdx.x / 16, rows, g.k, kt, row_of);
    few_quantize<XQ>(smem, raw, g.x, rows, g.k, kt, row_of);
    __syncthreads();
  }

  floatx16 acc[NB][TM];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[b][j][r] = 0.f;
  auto block = [&](const Part &p, int t) {
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      Fp8Frag<EXACT> x;
      float sa;
      if constexpr (XT == FEW_CODES) {
        // To operands through the wave's own LDS (its accesses run in order): chunk c of row r at c ^ ((r >> 1) & 7).
        uint8_t *q = smem + (wave * TM + j) * 4096;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i * 8 + (lane >> 3);
          *(intx4 *)(q + r * 128 + (((lane & 7) ^ ((r >> 1) & 7)) << 4)) = p.x[j][i];
        }
        const uint32_t off = (uint32_t)(col * 128 + (((2 * h) ^ ((col >> 1) & 7)) << 4));  // (chunk bits 0 and 2: ^ 16, ^ 64)
        x.set(0, *(const intx4 *)(q + off), *(const intx4 *)(q + (off ^ 16)));
        x.set(1, *(const intx4 *)(q + (off ^ 64)), *(const intx4 *)(q + (off ^ 80)));
        sa = p.sa[j];
      } else {
        const uint8_t *q = smem + (size_t)row[j] * few_row(kt) + t * 128 + h * 32;
        x.set(0, *(const intx4 *)q, *(const intx4 *)(q + 16));
        x.set(1, *(const intx4 *)(q + 64), *(const intx4 *)(q + 80));
        sa = s_as[row[j] * kt + t];
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        Fp8Frag<EXACT> a;
        a.set(0, p.w[b][0], p.w[b][1]);
        a.set(1, p.w[b][2], p.w[b][3]);
        const floatx16 c = fp8_product(a, x);
        const float s = sa * p.sw[b];
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[b][j][r] = __builtin_fmaf(c[r], s, acc[b][j][r]);
      }
    }
  };
  for (int it0 = 0; it0 < n_it; it0 += D)
    static_for<D>([&](auto d_c) {
      constexpr int d = decltype(d_c)::value;
      const int it = it0 + d;
      if (it < n_it) {
        block(ring[d], wk + kw * it);
        if (it + D < n_it) load(d_c, it + D);
      }
    });

  // Sums in LDS: [wave][output][quarter][half][column] of four values.
  floatx4 *red = (floatx4 *)(smem + (XT == FEW_CODES ? 0 : few_in(rows, kt)));
  if constexpr (XT == FEW_CODES) __syncthreads();
  const int cols = few_cols(TM == 1 ? rows : 32);
  if (col < cols)
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          red[((((wave * NB + b) * TM + j) * 4 + q) * 2 + h) * cols + col] =
              floatx4{acc[b][j][4 * q], acc[b][j][4 * q + 1], acc[b][j][4 * q + 2], acc[b][j][4 * q + 3]};
  __syncthreads();
  const int each = TM * 8 * cols;  // items of four values of a group
  for (int o = threadIdx.x; o < groups * each; o += FNW * 64) {
    const int gr = o / each, i = o - gr * each;
    const int c = i % cols, hq = i / cols, hh = hq & 1, q = (hq >> 1) & 3, j = hq >> 3;
    const int r = j * 32 + c, n = (nb0 + gr) * 32 + q * 8 + hh * 4;
    if (r >= rows || n >= g.n) continue;
    float v[NB][4];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      floatx4 sum = {0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < kw; ++k) {
        const floatx4 p = red[(((((gr * kw + k) * NB + b) * TM + j) * 4 + q) * 2 + hh) * cols + c];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += p[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[b][e] = sum[e];
    }
    if constexpr (MODE == FEW_GATE_UP) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[0][e] = fp8_silu_mul<EXACT>(v[0][e], v[1][e]);
    } else if constexpr (MODE == FEW_DOWN) {
      const float rw = g.row_w[row0 + r];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[0][e] *= rw;
    }
    fp8_store4(g.c, g.c_dtype, (row0 + r) * g.n + n, v[0], g.n - n);
  }
}

// The second product of tokens whose rows stand on their own, a tile each (few tokens: hardly two share an expert), with the
// sum over a token's experts: y (+)= Σ_p w_p · down_p(act_p), in the order of the rows, which is ascending expert id. A
// workgroup takes a token and a block of 32 outputs; its waves share the parts of K of all the token's experts. Row p is
// column p of the products, all others of its operand zeros, so that one accumulator holds them all.
//
// One token of a 30B-A3B layer, MI355X: 7.1 us (7.8 with eight waves), where the product and the combine of the lists' form
// take 4.7 each; the whole call 19.2 instead of 25.8. Bound by the trips to memory one behind the other: 12.6 MB.
constexpr int TNW = 16;  // waves
template <bool EXACT>
__global__ __launch_bounds__(TNW * 64) void fp8_token_kernel(const Fp8FewArgs g) {
  constexpr int D = 3;  // parts on the way, per wave
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int lane = lane_id(), col = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kt = g.kt, rows = g.top_k, n_nb = (g.n + 31) / 32, nb = blockIdx.x % n_nb;
  const int64_t t = blockIdx.x / n_nb, row0 = t * rows;
  const int expert = g.tiles[row0 + min(lane, rows - 1)].expert;  // lane p: row p's
  const float row_w = g.row_w[row0 + min(lane, rows - 1)];
  const int n_it = (rows * kt - wave + TNW - 1) / TNW;
  struct Part {
    intx4 w[4];
    float sw;
  } ring[D];
  auto load = [&](auto d_c, int it) {
    Part &r = ring[decltype(d_c)::value];
    const int u = wave + TNW * it, p = u / kt, k = u - p * kt, e = __builtin_amdgcn_readlane(expert, p);
    if (e < 0) return;
    const uint8_t *w = g.w + e * g.w_stride + ((int64_t)nb * kt + k) * 4096 + lane * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = *(const intx4 *)(w + i * 1024);
    r.sw = g.ws[e * g.ws_stride + (int64_t)(nb / 4) * kt + k];
  };
  const auto row_of = [&](int r) { return row0 + r; };
  dt_raw<RK_DTYPE_F32, 8> raw;
  few_load<RK_DTYPE_F32>(raw, g.x, threadIdx.x / 16, rows, g.k, kt, row_of);
  __builtin_amdgcn_sched_barrier(0);
  static_for<D>([&](auto d_c) {
    if (decltype(d_c)::value < n_it) load(d_c, decltype(d_c)::value);
  });
  __builtin_amdgcn_sched_barrier(0);
  const float *s_as = few_scales(smem, rows, kt);
  few_quantize<RK_DTYPE_F32, TNW>(smem, raw, g.x, rows, g.k, kt, row_of);
  __syncthreads();

  floatx16 acc = {};
  for (int it0 = 0; it0 < n_it; it0 += D)
    static_for<D>([&](auto d_c) {
      constexpr int d = decltype(d_c)::value;
      const int it = it0 + d;
      if (it < n_it) {
        const int u = wave + TNW * it, p = u / kt, k = u - p * kt;
        if (__builtin_amdgcn_readlane(expert, p) >= 0) {
          const intx4 zero = {0, 0, 0, 0};
          const bool mine = col == p;
          const uint8_t *q = smem + (size_t)p * few_row(kt) + k * 128 + h * 32;
          Fp8Frag<EXACT> a, x;
          x.set(0, mine ? *(const intx4 *)q : zero, mine ? *(const intx4 *)(q + 16) : zero);
          x.set(1, mine ? *(const intx4 *)(q + 64) : zero, mine ? *(const intx4 *)(q + 80) : zero);
          a.set(0, ring[d].w[0], ring[d].w[1]);
          a.set(1, ring[d].w[2], ring[d].w[3]);
          const floatx16 c = fp8_product(a, x);
          const float s = mine ? s_as[p * kt + k] * ring[d].sw : 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[r] = __builtin_fmaf(c[r], s, acc[r]);
        }
        if (it + D < n_it) load(d_c, it + D);
      }
    });

  // Sums over waves, [wave][quarter][half][row] of four outputs; then over rows.
  floatx4 *red = (floatx4 *)(smem + few_in(rows, kt));
  if (col < rows)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      red[((wave * 4 + q) * 2 + h) * rows + col] = floatx4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  __syncthreads();
  float *sums = (float *)smem;  // [row][32]
  for (int o = threadIdx.x; o < rows * 8; o += TNW * 64) {
    const int p = o % rows, hq = o / rows;
    floatx4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < TNW; ++k) sum += red[(k * 8 + hq) * rows + p];
    *(floatx4 *)(sums + p * 32 + (hq >> 1) * 8 + (hq & 1) * 4) = sum;
  }
  __syncthreads();
  const int n = nb * 32 + lane;
  if (wave > 0 || lane >= 32 || n >= g.n) return;
  const int64_t at = t * g.n + n;
  float y = g.accumulate ? dt_load_any(g.c, at, g.c_dtype) : 0.f;
  for (int p = 0; p < rows; ++p)
    if (__builtin_amdgcn_readlane(expert, p) >= 0) y += sums[p * 32 + lane] * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(row_w), p));
  if (g.c_dtype == RK_DTYPE_F32) dt_store<RK_DTYPE_F32>(g.c, at, y);
  else if (g.c_dtype == RK_DTYPE_F16) dt_store<RK_DTYPE_F16>(g.c, at, y);
  else dt_store<RK_DTYPE_BF16>(g.c, at, y);
}
static size_t token_smem(int rows, int kt) { return few_in(rows, kt) + (size_t)TNW * 128 * rows; }
// Rows of a token that fp8_token_kernel takes: columns of a product, in LDS.
bool rk_fp8_token_fits(int top_k, int kt) { return top_k <= 32 && token_smem(top_k, kt) <= 64 * 1024; }
hipError_t rk_launch_fp8_token(const Fp8FewArgs &g, int64_t s, bool exact, hipStream_t st) {
  if (!rk_fp8_token_fits(g.top_k, g.kt)) return hipErrorInvalidValue;
  auto kern = exact ? fp8_token_kernel<true> : fp8_token_kernel<false>;
  hipLaunchKernelGGL(kern, dim3((unsigned)(s * ((g.n + 31) / 32))), dim3(TNW * 64), token_smem(g.top_k, g.kt), st, g);
  return hipGetLastError();
}

// Rows that a workgroup can quantize into its LDS (x itself as input), and those that it can take as codes. Up to 32 rows of
// 64 KB of codes in all always fit: with K padded to 128, the scales and 16 bytes a row they are 65536·132/128 + 32·(132 + 16)
// bytes at most, and the sums behind them 32 KB.
bool rk_fp8_few_fits_x(int64_t m, int kt) { return m <= 32 && few_in((int)m, kt) <= 72320; }
// Where that is faster than a launch that quantizes once and a second one on codes: every workgroup takes 0.5 us for 32
// blocks of x. us so and in two launches, MI355X: 8 × 4096 × 2048 6.6 and 7.1, 16 × 4096 × 2048 8.8 and 7.2, 16 × 1024 ×
// 1024 5.7 and 6.2, 24 × 1024 × 1024 6.7 and 6.2, 4 × 4096 × 4096 8.1 and 8.8, 8 × 4096 × 4096 10.5 and 8.9.
bool rk_fp8_few_wants_x(int64_t m, int kt) { return m * kt <= 160; }
// Codes: while the grid is what is short, 32 outputs × 64 rows a workgroup, one per CU (two where the products are the
// slow exact ones). us here and on 64 × 128 tiles, MI355X, 16-bit results: 128 × 4096 × 4096 10.1 and 14.1, 256 × 2048 ×
// 2048 7.0 and 9.0, 192 × 4096 × 4096 15.5 and 14.5, 256 × 4096 × 1024 7.2 and 6.0; f32: 512 × 2048 × 2048 12.0 and 13.6,
// 768 × 2048 × 2048 18 and 14. Up to 32 rows a wave has one column block, and the weight streams: 32 × 16384 × 2048 9.7 and 10.2.
bool rk_fp8_few_fits_codes(int64_t m, int64_t n, bool exact, int num_cus) {
  return m <= 32 || (n + 31) / 32 * ((m + 63) / 64) <= (exact ? 2 : 1) * (int64_t)num_cus;
}
// Rows of an expert tile that a workgroup has LDS for: a power of two of at most 32.
int rk_fp8_few_rows(int kt) {
  int rows = 32;
  while (rows > 1 && few_smem(0, 2, 1, rows, kt) > 160 * 1024) rows /= 2;
  return rows;
}

template <int XT, int MODE, bool EXACT, int TM>
static hipError_t launch_few(Fp8FewArgs g, int rows, int n_tiles, hipStream_t st) {
  constexpr int NOUT = (MODE == FEW_GATE_UP ? 2 : 1) * TM;
  auto kern = fp8_few_kernel<XT, MODE, EXACT, TM>;
  static bool attr_set = false;
  if (!attr_set) {
    hipError_t e = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return e;
    attr_set = true;
  }
  const size_t smem = few_smem(XT, NOUT, TM, TM == 1 ? rows : 32, g.kt);
  if (smem > 160 * 1024) return hipErrorInvalidValue;
  // Blocks side by side in a workgroup: as many as leave a workgroup per CU, and a wave at most eight parts of K. Whole
  // calls on a 30B-A3B layer, MI355X, with G of the first product's blocks and D of the second's: 64 tokens 171 us with 1
  // and 1, 135 with 4 and 8; one token 28.2 with 1 and 1, 25.5 with 1 and 2, 25.9 with 2 and 4. From codes a workgroup is a
  // round of its CU: also where that leaves fewer (384 × 2048 × 2048 11.4 and 9.6 us).
  const int64_t n_nb = (g.n + 31) / 32;
  const auto wgs = [&](int groups) { return (n_nb + groups - 1) / groups * n_tiles; };
  g.groups = 1;
  while (g.groups < FNW && (XT == FEW_CODES ? wgs(g.groups) > g.num_cus : wgs(2 * g.groups) >= g.num_cus) && g.kt * 2 * g.groups <= 8 * FNW)
    g.groups *= 2;
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs(g.groups)), dim3(FNW * 64), smem, st, g);
  return hipGetLastError();
}

hipError_t rk_launch_fp8_few_gate_up(const Fp8FewArgs &g, int x_dtype, int tile_rows, int n_tiles, bool exact, hipStream_t st) {
#define RK_FEW(XT) (exact ? launch_few<XT, FEW_GATE_UP, true, 1>(g, tile_rows, n_tiles, st) : launch_few<XT, FEW_GATE_UP, false, 1>(g, tile_rows, n_tiles, st))
  switch (x_dtype) {
    case RK_DTYPE_F32: return RK_FEW(RK_DTYPE_F32);
    case RK_DTYPE_F16: return RK_FEW(RK_DTYPE_F16);
    default: return RK_FEW(RK_DTYPE_BF16);
  }
#undef RK_FEW
}
hipError_t rk_launch_fp8_few_down(const Fp8FewArgs &g, int tile_rows, int n_tiles, bool exact, hipStream_t st) {
  return exact ? launch_few<RK_DTYPE_F32, FEW_DOWN, true, 1>(g, tile_rows, n_tiles, st)
               : launch_few<RK_DTYPE_F32, FEW_DOWN, false, 1>(g, tile_rows, n_tiles, st);
}

hipError_t rk_launch_fp8_few(const Fp8FewArgs &g, int x_dtype, bool exact, hipStream_t st) {
  // Column blocks (32 rows) of a call, a wave's share of them: two where one each would be more than a round of workgroups
  // (with four the registers do not do). They read the weight once per share, which the caches serve.
  const int cb = x_dtype == FEW_CODES ? (g.m + 31) / 32 : 1, n_nb = (g.n + 31) / 32;
  const int tm = (int64_t)n_nb * cb > g.num_cus ? min(cb, 2) : 1;
  const int tiles = (cb + tm - 1) / tm;
#define RK_FEW(XT, TM) \
  (exact ? launch_few<XT, FEW_DENSE, true, TM>(g, g.m, tiles, st) : launch_few<XT, FEW_DENSE, false, TM>(g, g.m, tiles, st))
  switch (x_dtype) {
    case RK_DTYPE_F32: return RK_FEW(RK_DTYPE_F32, 1);
    case RK_DTYPE_F16: return RK_FEW(RK_DTYPE_F16, 1);
    case RK_DTYPE_BF16: return RK_FEW(RK_DTYPE_BF16, 1);
  }
  return tm == 1 ? RK_FEW(FEW_CODES, 1) : RK_FEW(FEW_CODES, 2);
#undef RK_FEW
}
