// Block-scaled fp8 experts on many rows: the two grouped products over tiles of bucket rows, on the K loop of the dense
// product (fp8_tile.hpp). Few rows a tile: fp8_few.hip.
//
//   gate|up  rows gathered by their tokens; gate and up blocks of 32 weight rows lie in turns, so that a wave holds the gate
//            and the up value of an output in one lane. A workgroup's 256 weight rows are 128 outputs: a whole block of the
//            next product's activations, which it quantizes itself. act goes out as codes and scales, a quarter of f32's bytes
//            and with no pass of its own.
//   down     bucket rows as they lie, times their router weight, to rows that the combine sums per token.
#include "fp8_tile.hpp"
#include "kernels.hpp"

// Tile and column of a workgroup: tile t on XCD t mod 8, all its columns there, sharing its rows in that XCD's L2. Tiles
// listed for more rows than the workgroup takes are `parts` tiles.
__device__ __forceinline__ bool moe_fp8_place(const Fp8MoeArgs &g, int bm, int n_col, MoeTile &tile, int &nc) {
  const int jb = blockIdx.x / 8, t = blockIdx.x % 8 + 8 * (jb / n_col), parts = g.tile_rows / bm;
  if (t >= g.n_tiles * parts) return false;
  tile = g.tiles[t / parts];
  const int first = t % parts * bm;
  tile.row0 += first;
  tile.rows = min(tile.rows - first, bm);
  nc = jb % n_col;
  return tile.rows > 0 && tile.expert >= 0;
}

template <class T>
__global__ __launch_bounds__(T::NT, 2) void moe_fp8_gate_up_kernel(const Fp8MoeArgs g) {
  static_assert(T::BN == 256 && T::TN % 2 == 0, "128 outputs, gate and up in one wave");
  constexpr int P = T::TN / 2;  // gate|up pairs of a wave
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  MoeTile tile;
  int nc;
  const int KT = g.kt, ib = (g.n + 127) / 128;
  if (!moe_fp8_place(g, T::BM, ib, tile, nc)) return;
  const uint8_t *w = g.w + (int64_t)tile.expert * g.w_stride + (int64_t)nc * 8 * KT * 4096;
  const float *ws = g.ws + (int64_t)tile.expert * 2 * ib * KT;
  T t;
  t.run(smem, g.a, (int64_t)g.n_tok * g.k, g.as, (int64_t)g.n_tok * KT * 4,
        [&](int r) -> int64_t { return r < tile.rows ? (int64_t)g.tok[tile.row0 + r] : -1; }, tile.rows, w, 8, ws,
        (int64_t)2 * ib * KT * 4, [&](int b) { return (int64_t)((b & 1) * ib + nc) * KT; }, g.k, KT);

  // act in place of the gate; the largest of a row's 128 over the lane's two halves and the workgroup's waves.
  const int tid = fresh_tid(), col = tid & 31, h = (tid >> 5) & 1;
  const int wave = tid >> 6, wm = wave / T::WN, wn = wave % T::WN;
  float *s_max = (float *)smem;                                         // [WN][BM]
  uint8_t *s_out = smem + T::WN * T::BM * 4;                            // [BM][144]: a row's codes
  constexpr int ROW = 144;
  static_assert(T::WN * T::BM * 4 + T::BM * ROW <= T::SMEM, "epilogue LDS");
  float amax[T::TM];
#pragma unroll
  for (int j = 0; j < T::TM; ++j) {
    amax[j] = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float v = fp8_silu_mul<T::EXACT>(t.acc[2 * p][j][r], t.acc[2 * p + 1][j][r]);
        t.acc[2 * p][j][r] = v;
        amax[j] = fmaxf(amax[j], fabsf(v));
      }
    amax[j] = fmaxf(amax[j], __shfl_xor(amax[j], 32));
    if (h == 0) s_max[wn * T::BM + wm * T::WTM + j * 32 + col] = amax[j];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < T::TM; ++j) {
    const int r = wm * T::WTM + j * 32 + col;
    float m = 0.f;
#pragma unroll
    for (int x = 0; x < T::WN; ++x) m = fmaxf(m, s_max[x * T::BM + r]);
    const float s = fp8_scale(m);
    const Fp8Div div(s);
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const floatx16 &v = t.acc[2 * p][j];
        *(uint32_t *)(s_out + r * ROW + (wn * P + p) * 32 + q * 8 + h * 4) =
            fp8_codes4(div(v[4 * q]), div(v[4 * q + 1]), div(v[4 * q + 2]), div(v[4 * q + 3]));
      }
    if (wn == 0 && h == 0 && r < tile.rows) g.out_s[((int64_t)tile.row0 + r) * ib + nc] = s;
  }
  __syncthreads();
  for (int c = tid; c < tile.rows * 8; c += T::NT) {
    const int r = c >> 3, at = (c & 7) * 16;
    *(uintx4 *)((uint8_t *)g.out + ((int64_t)tile.row0 + r) * ib * 128 + nc * 128 + at) = *(const uintx4 *)(s_out + r * ROW + at);
  }
}

// ROWS16: the weighted rows as fp16 under scales, for bf16 results; f32 otherwise.
template <class T, bool ROWS16>
__global__ __launch_bounds__(T::NT, 2) void moe_fp8_down_kernel(const Fp8MoeArgs g) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  MoeTile tile;
  int nc;
  const int KT = g.kt, nblk = (g.n + 127) / 128 * 4;
  if (!moe_fp8_place(g, T::BM, (g.n + T::BN - 1) / T::BN, tile, nc)) return;
  const int nb0 = nc * (T::BN / 32), n0 = nc * T::BN;
  const float *ws = g.ws + (int64_t)tile.expert * (nblk / 4) * KT;
  T t;
  t.run(smem, g.a + (int64_t)tile.row0 * KT * 128, (int64_t)tile.rows * KT * 128, g.as + (int64_t)tile.row0 * KT, (int64_t)tile.rows * KT * 4,
        [&](int r) -> int64_t { return r < tile.rows ? r : -1; }, tile.rows, g.w + (int64_t)tile.expert * g.w_stride + (int64_t)nb0 * KT * 4096,
        nblk - nb0, ws, (int64_t)(nblk / 4) * KT * 4, [&](int b) { return (int64_t)min((nb0 + b) / 4, nblk / 4 - 1) * KT; }, KT * 128, KT);
  // Rows times their router weight, in f32 for f32 and fp16 results: an fp16 row's rounding is as large as the result's own, and
  // larger where experts cancel. In front of bf16 results (2^-8 of a result) fp16 rows, under a power of two per row and wave
  // (T::WTN outputs) that takes the largest to [2^14, 2^15): 2^-11 of a term, and below 2^-28 of the largest 2^-39 of that,
  // for half of the bytes (8192 tokens of a 64-expert layer, MI355X: this product and the combine 261 us, with f32 rows 351; the
  // layer in fp16 1053 us, and 974 with fp16 rows).
  float *const to = (float *)g.out + (int64_t)tile.row0 * g.n + n0;
  const int tid = fresh_tid(), col = tid & 31, h = (tid >> 5) & 1;
  const int wave = tid >> 6, wm = wave / T::WN, wn = wave % T::WN;
  float rw[T::TM];
#pragma unroll
  for (int j = 0; j < T::TM; ++j) {
    const int r = wm * T::WTM + j * 32 + col;
    rw[j] = r < tile.rows ? g.row_w[tile.row0 + r] : 0.f;
    if constexpr (ROWS16) {
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < T::TN; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          t.acc[i][j][e] *= rw[j];
          amax = fmaxf(amax, fabsf(t.acc[i][j][e]));
        }
      amax = fmaxf(amax, __shfl_xor(amax, 32));
      if (amax == INFINITY) {  // the largest of the finite ones: an infinite one needs no scale
        amax = 0.f;
#pragma unroll
        for (int i = 0; i < T::TN; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float v = fabsf(t.acc[i][j][e]);
            amax = fmaxf(amax, v < INFINITY ? v : 0.f);
          }
        amax = fmaxf(amax, __shfl_xor(amax, 32));  // (both lanes of a row are here)
      }
      // exponent of the largest; nothing to scale in rows of zeros
      const int x = amax > 0.f ? max((int)(__float_as_uint(amax) >> 23) - 127 - 14, -100) : 0;
      rw[j] = ldexpf(1.f, -x);
      if (h == 0 && r < tile.rows && n0 + wn * T::WTN < g.n)
        g.out_s[((int64_t)tile.row0 + r) * ((g.n + T::WTN - 1) / T::WTN) + (n0 + wn * T::WTN) / T::WTN] = ldexpf(1.f, x);
    }
  }
  const auto value = [&](int i, int j, int r) { return t.acc[i][j][r] * rw[j]; };
  if constexpr (ROWS16) {
    fp8_store_tile<T, RK_DTYPE_F16>(smem, value, (uint16_t *)g.out + (int64_t)tile.row0 * g.n + n0, g.n, tile.rows, g.n - n0);
  } else if constexpr (T::BM * T::BN * 4 <= T::SMEM) {
    fp8_store_tile<T, RK_DTYPE_F32>(smem, value, to, g.n, tile.rows, g.n - n0);
  } else {
#pragma unroll
    for (int j = 0; j < T::TM; ++j) {
      const int r = wm * T::WTM + j * 32 + col;
      if (r >= tile.rows) continue;
#pragma unroll
      for (int i = 0; i < T::TN; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = wn * T::WTN + i * 32 + q * 8 + h * 4;
          if (n0 + n < g.n)  // (a multiple of 16 outputs)
            *(floatx4 *)(to + (int64_t)r * g.n + n) = floatx4{value(i, j, 4 * q), value(i, j, 4 * q + 1), value(i, j, 4 * q + 2), value(i, j, 4 * q + 3)};
        }
    }
  }
}

template <class T, bool GU, bool ROWS16 = false>
static hipError_t launch_moe_fp8(const Fp8MoeArgs &g, hipStream_t st) {
  void (*kern)(const Fp8MoeArgs);
  if constexpr (GU) kern = moe_fp8_gate_up_kernel<T>;
  else kern = moe_fp8_down_kernel<T, ROWS16>;
  static bool attr_set = false;
  if (!attr_set) {
    hipError_t e = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
    if (e != hipSuccess) return e;
    attr_set = true;
  }
  const int n_col = GU ? (g.n + 127) / 128 : (g.n + T::BN - 1) / T::BN;
  hipLaunchKernelGGL(kern, dim3((unsigned)((g.n_tiles * (g.tile_rows / T::BM) + 7) / 8 * 8 * n_col)), dim3(T::NT), T::SMEM, st, g);
  return hipGetLastError();
}

template <bool GU>
static hipError_t launch_moe_fp8_any(const Fp8MoeArgs &g, bool exact, hipStream_t st) {
  if (g.tile_rows != 128 && g.tile_rows != 256) return hipErrorInvalidValue;
  // 256 rows: fewer passes over the rows' and the weights' bytes, 64 × 128 a wave. 128 rows stream weights more than they
  // compute: a third stage on the way for the first product; tiles of 128 outputs, two a CU, for the second, whose K is short.
  // 1024 tokens of a 30B-A3B layer, MI355X: first product 94 us (102 with two stages; its weights take 85), second 56 (58 with
  // 256 outputs and three stages, 61 with two, 72 with 64 rows; its weights take 43).
  if constexpr (GU) {
    if (exact) return launch_moe_fp8<Fp8Tile<128, 256, 2, 4, 3, true>, GU>(g, st);
    if (g.tile_rows == 256) return launch_moe_fp8<Fp8Tile<256, 256, 4, 2, 2, false>, GU>(g, st);
    return launch_moe_fp8<Fp8Tile<128, 256, 2, 4, 3, false>, GU>(g, st);
  } else {
    const bool rows16 = g.out_s != nullptr;
    if (exact) return rows16 ? hipErrorInvalidValue : launch_moe_fp8<Fp8Tile<128, 256, 2, 4, 2, true>, GU>(g, st);
    using Large = Fp8Tile<256, 256, 4, 2, 2, false>;
    using Small = Fp8Tile<128, 128, 2, 2, 2, false>;
    if (g.tile_rows == 256) return rows16 ? launch_moe_fp8<Large, GU, true>(g, st) : launch_moe_fp8<Large, GU>(g, st);
    return rows16 ? launch_moe_fp8<Small, GU, true>(g, st) : launch_moe_fp8<Small, GU>(g, st);
  }
}
hipError_t rk_launch_moe_fp8_gate_up(const Fp8MoeArgs &g, bool exact, hipStream_t st) {
  return launch_moe_fp8_any<true>(g, exact, st);
}
// Outputs under one scale of the second product's fp16 rows.
int rk_moe_fp8_down_group(int tile_rows) { return tile_rows == 256 ? 128 : 64; }
hipError_t rk_launch_moe_fp8_down(const Fp8MoeArgs &g, bool exact, hipStream_t st) {
  return launch_moe_fp8_any<false>(g, exact, st);
}
