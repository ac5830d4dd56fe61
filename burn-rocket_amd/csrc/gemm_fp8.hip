// Products of many rows with a block-scaled fp8 weight (e4m3 codes, one f32 scale per 128 × 128 block of the weight and per
// row and 128 values of the activations):
//
//   c[m, n] = Σ_b as[m, b] · ws[n / 128, b] · P_b[m, n],  P_b the product of block b's codes,
//
// summed in f32 in block order (fp8_tile.hpp).
#include "fp8_tile.hpp"
#include "kernels.hpp"

template <class T>
__global__ __launch_bounds__(T::NT, 2) void gemm_fp8_kernel(const Fp8GemmArgs g, int tiles_m, int tiles_n, int group_m) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  int tm, tn;
  tile_coords(xcd_remap(blockIdx.x, gridDim.x), tiles_m, tiles_n, group_m, tm, tn);
  const int64_t m0 = (int64_t)tm * T::BM;
  const int n0 = tn * T::BN, KT = g.kt;
  const int64_t left = g.m - m0;
  const int rows = (int)min<int64_t>(left, T::BM);
  const int nblk = (g.n + 127) / 128 * 4;
  T t;
  t.run(smem, g.a + m0 * g.k, left * g.k, g.as + m0 * KT, left * KT * 4, [&](int r) -> int64_t { return r < rows ? r : -1; }, rows,
        g.w + (int64_t)(n0 / 32) * KT * 4096, nblk - n0 / 32,
        g.ws, (int64_t)(nblk / 4) * KT * 4, [&](int b) { return (int64_t)min((n0 / 32 + b) / 4, nblk / 4 - 1) * KT; }, g.k, KT);

  const auto value = [&](int i, int j, int r) { return t.acc[i][j][r]; };
  const auto out = [&](int es) { return (uint8_t *)g.c + (m0 * g.n + n0) * es; };
  if constexpr (T::EXACT)
    if (g.c_dtype == RK_DTYPE_F32) return fp8_store_tile<T, RK_DTYPE_F32>(smem, value, out(4), g.n, rows, g.n - n0);
  if (g.c_dtype == RK_DTYPE_F16) fp8_store_tile<T, RK_DTYPE_F16>(smem, value, out(2), g.n, rows, g.n - n0);
  else fp8_store_tile<T, RK_DTYPE_BF16>(smem, value, out(2), g.n, rows, g.n - n0);
}

template <class T>
static hipError_t launch_fp8(const Fp8GemmArgs &g, hipStream_t st) {
  auto kern = gemm_fp8_kernel<T>;
  static bool attr_set = false;
  if (!attr_set) {
    hipError_t e = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
    if (e != hipSuccess) return e;
    attr_set = true;
  }
  const int tm = (int)((g.m + T::BM - 1) / T::BM), tn = (g.n + T::BN - 1) / T::BN;
  hipLaunchKernelGGL(kern, dim3((unsigned)tm * tn), dim3(T::NT), T::SMEM, st, g, tm, tn, rk_knob("RK_TILE_GROUP_M", 4));
  return hipGetLastError();
}

// f32 results take the exact products.
hipError_t rk_launch_gemm_fp8(const Fp8GemmArgs &g, bool exact, hipStream_t st) {
  if (!exact && g.c_dtype == RK_DTYPE_F32) return hipErrorInvalidValue;
  const auto tiles = [&](int bm, int bn) { return (int64_t)((g.m + bm - 1) / bm) * ((g.n + bn - 1) / bn); };
  const auto rounds = [&](int64_t n, int64_t at_once) { return (n + at_once - 1) / at_once; };
  // At most one and a half 64 × 128 tiles per CU: a round of them ends sooner than one of 128 × 128 would. us so and with these,
  // MI355X, 16-bit results: 2048 × 1024 × 4096 16.6 and 22, 512 × 4096 × 4096 16.0 and 21.8, 1024 × 4096 × 4096 (two per CU)
  // 27.7 and 25.2, 3633 × 1024 × 2560 (1.8) 17.9 and 17.0; f32: 2048 × 1024 × 4096 24 and 35, 4096 × 1024 × 4096 39 and 40.
  // (Fp8Tile with these sizes, weights through LDS: the six 18, 18, 27.4, 18.4; 30, 43; 4096 × 4096 × 4096 in f32 131 where
  // this is 111.)
  const bool small = 2 * tiles(64, 128) <= 3 * g.num_cus;
  if (exact) return small ? launch_fp8<Fp8Flow<2, 3, true>>(g, st) : launch_fp8<Fp8Flow<4, 3, true>>(g, st);
  if (small) return launch_fp8<Fp8Flow<2, 3, false>>(g, st);
  // 256 × 256 where its rounds, one tile a CU, are less than two thirds of those of 128 × 128, two a CU: a round of them
  // takes 47 to 60 us at K = 4096, one of these 34 to 38 (2560 × 4096: 54 and 63; 2048 × 4096: 51 and 38; 4608 × 4096: 100
  // and 96).
  if (3 * rounds(tiles(256, 256), g.num_cus) < 2 * rounds(tiles(128, 128), 2 * g.num_cus)) return launch_fp8<Fp8Tile<256, 256, 4, 2, 2, false>>(g, st);
  return launch_fp8<Fp8Flow<4, 3, false>>(g, st);
}
