// Products of few rows with a block-scaled fp8 weight: decode steps of a dense layer, and expert tiles of at most 32 rows.
//
// These are bound by the weight's bytes and, below a few MB, by latency: no wave may wait for another while it streams. A
// workgroup takes one 32-row block of the weight (of an expert's first product: a gate and its up block) and its waves split
// K: wave w reads the 4 KB blocks w, w + 8, .. of its row block in four 1 KB pieces, some of them ahead, straight into the
// registers that a 32 × 32 product reads them from. The partial sums meet in LDS at the end, in wave order.
//
// The rows (32 columns of the products, most of them empty in a decode step) come as x itself: the workgroup quantizes them
// into LDS while its first weights are on the way, so that a layer is one launch; or, where they do not fit LDS, as codes
// that each wave reads from the caches, up to four column blocks a wave.
#include "fp8.hpp"
#include "kernels.hpp"

namespace {
enum { FEW_DENSE = 0, FEW_GATE_UP = 1, FEW_DOWN = 2 };
constexpr int FNW = 8;  // waves, the split of K
constexpr int FEW_CODES = 3;  // x's type: codes and scales

// Bytes of a quantized row in LDS: 16 more than its codes, which spreads the rows over the banks.
__host__ __device__ constexpr int few_row(int kt) { return kt * 128 + 16; }
template <int XT, int NOUT>
size_t few_smem(int rows, int kt) {
  const size_t red = (size_t)FNW * NOUT * 4096;
  const size_t in = XT == FEW_CODES ? 0 : (size_t)rows * (few_row(kt) + kt * 4);
  return red > in ? red : in;
}
}  // namespace

template <int XT, int MODE, bool EXACT, int TM>
__global__ __launch_bounds__(FNW * 64, 2) void fp8_few_kernel(const Fp8FewArgs g) {
  constexpr int NB = MODE == FEW_GATE_UP ? 2 : 1;  // weight blocks
  constexpr int D = NB == 2 || TM > 2 ? 2 : 4;     // blocks of K on the way, per wave
  static_assert(XT == FEW_CODES || TM == 1, "x in LDS: one column block");
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int lane = lane_id(), col = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kt = g.kt;
  // (a tile's workgroups one behind the other: they share its rows)
  const int n_nb = (g.n + 31) / 32, nb = blockIdx.x % n_nb;
  int rows = g.m;
  int64_t row0 = 0;
  const uint8_t *w = g.w;
  const float *ws = g.ws;
  if constexpr (MODE != FEW_DENSE) {
    const MoeTile tile = g.tiles[blockIdx.x / n_nb];
    if (tile.rows <= 0 || tile.expert < 0) return;
    rows = tile.rows;
    row0 = tile.row0;
    w += (int64_t)tile.expert * g.w_stride;
    ws += (int64_t)tile.expert * g.ws_stride;
  }

  // Weight blocks of this workgroup: consecutive in the layout. Scales: of the gate rows, then of the up rows.
  const uint8_t *wb = w + (int64_t)nb * NB * kt * 4096 + lane * 16;
  const float *wsb = ws + (int64_t)(nb / 4) * kt;
  intx4 ring[D][NB][4];
  auto load = [&](auto d_c, int t) {
    constexpr int d = decltype(d_c)::value;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) ring[d][b][i] = *(const intx4 *)(wb + ((int64_t)b * kt + t) * 4096 + i * 1024);
  };
  const int n_it = (kt - wave + FNW - 1) / FNW;  // (may be 0)
  static_for<D>([&](auto d_c) {
    if (decltype(d_c)::value < n_it) load(d_c, wave + FNW * decltype(d_c)::value);
  });

  // x to codes in LDS, [row][few_row], scales [row][kt] behind them.
  float *s_as = (float *)(smem + (size_t)rows * few_row(kt));
  if constexpr (XT != FEW_CODES) {
    const int sub = threadIdx.x & 15;
    for (int b = threadIdx.x / 16; b < rows * kt; b += FNW * 4) {
      const int r = b / kt, at = b - r * kt, c = at * 128 + sub * 8;
      const int64_t src = MODE == FEW_GATE_UP ? (int64_t)min(g.tok[row0 + r], g.n_tok - 1) : row0 + r;
      float v[8];
      if (c < g.k) {
        if constexpr (XT == RK_DTYPE_F32) {
          dt_load_vec<XT, 4>(g.x, src * g.k + c, v);
          dt_load_vec<XT, 4>(g.x, src * g.k + c + 4, v + 4);
        } else {
          dt_load_vec<XT, 8>(g.x, src * g.k + c, v);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
      }
      float amax = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(v[e]));
#pragma unroll
      for (int d = 1; d < 16; d *= 2) amax = fmaxf(amax, __shfl_xor(amax, d));
      const float s = fp8_scale(amax);
      const Fp8Div div(s);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = div(v[e]);
      *(uintx2 *)(smem + (size_t)r * few_row(kt) + c) =
          uintx2{fp8_codes4(v[0], v[1], v[2], v[3]), fp8_codes4(v[4], v[5], v[6], v[7])};
      if (sub == 0) s_as[r * kt + at] = s;
    }
    __syncthreads();
  }

  floatx16 acc[NB][TM];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[b][j][r] = 0.f;
  // Columns past the last row repeat it: they are not stored.
  int row[TM];
#pragma unroll
  for (int j = 0; j < TM; ++j) row[j] = min(j * 32 + col, rows - 1);
  const uint8_t *codes = (const uint8_t *)g.x;
  auto block = [&](auto d_c, int t) {
    constexpr int d = decltype(d_c)::value;
    Fp8Frag<EXACT> a[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      a[b].set(0, ring[d][b][0], ring[d][b][1]);
      a[b].set(1, ring[d][b][2], ring[d][b][3]);
    }
    float sw[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) sw[b] = wsb[(int64_t)b * g.up_scales + t];
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      Fp8Frag<EXACT> x;
      float sa;
      intx4 c[4];
      if constexpr (XT == FEW_CODES) {
        const int64_t r = row0 + row[j];
        const uint8_t *p = codes + r * g.k + t * 128 + h * 32;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = (i >> 1) * 64 + (i & 1) * 16;
          c[i] = t * 128 + h * 32 + at < g.k ? *(const intx4 *)(p + at) : intx4{0, 0, 0, 0};
        }
        sa = g.as[r * kt + t];
      } else {
        const uint8_t *p = smem + (size_t)row[j] * few_row(kt) + t * 128 + h * 32;
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = *(const intx4 *)(p + (i >> 1) * 64 + (i & 1) * 16);
        sa = s_as[row[j] * kt + t];
      }
      x.set(0, c[0], c[1]);
      x.set(1, c[2], c[3]);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const floatx16 p = fp8_product(a[b], x);
        const float s = sa * sw[b];
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[b][j][r] = __builtin_fmaf(p[r], s, acc[b][j][r]);
      }
    }
  };
  for (int it0 = 0; it0 < n_it; it0 += D)
    static_for<D>([&](auto d_c) {
      const int it = it0 + decltype(d_c)::value;
      if (it < n_it) {
        block(d_c, wave + FNW * it);
        if (it + D < n_it) load(d_c, wave + FNW * (it + D));
      }
    });

  // The waves' sums: [wave][output][quarter][lane] of four values.
  __syncthreads();
  floatx4 *red = (floatx4 *)smem;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        red[(((wave * NB + b) * TM + j) * 4 + q) * 64 + lane] =
            floatx4{acc[b][j][4 * q], acc[b][j][4 * q + 1], acc[b][j][4 * q + 2], acc[b][j][4 * q + 3]};
  __syncthreads();
  const bool whole = (g.n & 3) == 0;
  for (int o = threadIdx.x; o < TM * 256; o += FNW * 64) {
    const int l = o & 63, q = (o >> 6) & 3, j = o >> 8;
    const int r = j * 32 + (l & 31);
    if (r >= rows) continue;
    float v[NB][4];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < FNW; ++k) {
        const floatx4 p = red[(((k * NB + b) * TM + j) * 4 + q) * 64 + l];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += p[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[b][e] = sum[e];
    }
    const int n = nb * 32 + q * 8 + (l >> 5) * 4;
    if constexpr (MODE == FEW_GATE_UP) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[0][e] = fp8_silu_mul<EXACT>(v[0][e], v[1][e]);
    } else if constexpr (MODE == FEW_DOWN) {
      const float rw = g.row_w[row0 + r];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[0][e] *= rw;
    }
    fp8_store4(g.c, g.c_dtype, (row0 + r) * g.n + n, v[0], g.n - n, whole);
  }
}

// Rows that a workgroup can quantize into its LDS (x itself as input), and those that it can take as codes.
bool rk_fp8_few_fits_x(int64_t m, int kt) { return m <= 32 && few_smem<0, 1>((int)m, kt) <= 64 * 1024; }
bool rk_fp8_few_fits_codes(int64_t m) { return m <= 128; }

template <int XT, int MODE, bool EXACT, int TM>
static hipError_t launch_few(const Fp8FewArgs &g, int rows, int n_tiles, hipStream_t st) {
  constexpr int NOUT = (MODE == FEW_GATE_UP ? 2 : 1) * TM;
  auto kern = fp8_few_kernel<XT, MODE, EXACT, TM>;
  static bool attr_set = false;
  if (!attr_set) {
    hipError_t e = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return e;
    attr_set = true;
  }
  const size_t smem = few_smem<XT, NOUT>(rows, g.kt);
  if (smem > 160 * 1024) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kern, dim3((unsigned)((int64_t)(g.n + 31) / 32 * n_tiles)), dim3(FNW * 64), smem, st, g);
  return hipGetLastError();
}

// Rows of an expert tile that a workgroup has LDS for: a power of two of at most 32.
int rk_fp8_few_rows(int kt) {
  int rows = 32;
  while (rows > 1 && few_smem<0, 2>(rows, kt) > 160 * 1024) rows /= 2;
  return rows;
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
#define RK_FEW(XT, TM) (exact ? launch_few<XT, FEW_DENSE, true, TM>(g, g.m, 1, st) : launch_few<XT, FEW_DENSE, false, TM>(g, g.m, 1, st))
  switch (x_dtype) {
    case RK_DTYPE_F32: return RK_FEW(RK_DTYPE_F32, 1);
    case RK_DTYPE_F16: return RK_FEW(RK_DTYPE_F16, 1);
    case RK_DTYPE_BF16: return RK_FEW(RK_DTYPE_BF16, 1);
  }
  return g.m <= 32 ? RK_FEW(FEW_CODES, 1) : g.m <= 64 ? RK_FEW(FEW_CODES, 2) : RK_FEW(FEW_CODES, 4);
#undef RK_FEW
}
