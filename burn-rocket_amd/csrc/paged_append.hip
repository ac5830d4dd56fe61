// K and V of new tokens into a paged cache, with the attention prologue on the
// way: RMSNorm over the head dim (optional) and rotate-half RoPE of the q and k
// heads of a fused q|k|v projection, q to its own rows, k and v to the slots that
// the tokens' sequences hold.
//
//   y = x · w / sqrt(Σx²/D + eps)
//   o[j] = y[j]·cos[j] − y[j + D/2]·sin[j],  o[j + D/2] = y[j + D/2]·cos[j] + y[j]·sin[j]
//
// All in f32 and rounded once, at the store (rk_qk_norm_rope_dev rounds y as well,
// as the separate ops it stands for do). Bound by memory: a row is read once and
// written once. A lane takes the same CV values of both halves of a head, so that
// the rotation needs no other lane and each lane has two loads in flight per
// row; D/(2·CV) lanes make a row (rounded up to a power of two), the sum of
// squares is a butterfly over them. V heads take the same lanes and are copied.
// MI355X: six prompts of 900 to 2400 tokens, 32/4 heads of 128, norm, bf16: 30.8 us (184 MB,
// 6.0 TB/s); 48 rows of 16/8 heads of 128 3.4 us, which is a launch and two trips to memory.
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"

namespace {
struct AppendGeom {
  int rows;       // tokens × (q + k + v heads)
  int lpr_log2;   // lanes per row
};
}  // namespace

template <int DT, int CT, int CV>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a, AppendGeom ag) {
  const int lane = threadIdx.x & 63, lpr = 1 << ag.lpr_log2, li = lane & (lpr - 1);
  const int heads = a.n_head + 2 * a.n_kv_heads, half = a.head_dim / 2;
  const int row = (int)(blockIdx.x * (256u >> ag.lpr_log2) + (threadIdx.x >> ag.lpr_log2));
  if (row - (lane >> ag.lpr_log2) >= ag.rows) return;  // no row of this wave
  const int t = (int)((uint32_t)row / (uint32_t)heads), hh = row - t * heads;
  const int j = li * CV;
  bool live = row < ag.rows && j < half;
  dt_raw<DT, CV> x0{}, x1{}, w0{}, w1{};
  dt_raw<CT, CV> c{}, s{};
  SeqTok tk{};
  const bool rot = hh < a.n_head + a.n_kv_heads;
  const void *w = hh < a.n_head ? a.q_norm_w : a.k_norm_w;
  if (live) {
    tk = a.toks[t];
    live = tk.page >= 0;  // a captured launch has room for more tokens than a batch may have
  }
  if (live) {
    const int64_t at = (int64_t)t * a.row_stride + (int64_t)hh * a.head_dim + j;
    dt_load_raw<DT, CV>(a.qkv, at, x0);
    dt_load_raw<DT, CV>(a.qkv, at + half, x1);
    if (rot) {
      if (w) {
        dt_load_raw<DT, CV>(w, j, w0);
        dt_load_raw<DT, CV>(w, j + half, w1);
      }
      dt_load_raw<CT, CV>(a.cos, (int64_t)tk.pos * half + j, c);
      dt_load_raw<CT, CV>(a.sin, (int64_t)tk.pos * half + j, s);
    }
  }
  float f0[CV], f1[CV];
  dt_decode_raw<DT, CV>(x0, f0);
  dt_decode_raw<DT, CV>(x1, f1);
  if (w) {  // the lanes of a row have the same w; all take part in its sum
    float acc = 0.f;
#pragma unroll
    for (int e = 0; e < CV; ++e) acc += f0[e] * f0[e] + f1[e] * f1[e];
    for (int off = lpr >> 1; off >= 1; off >>= 1) acc += __shfl_xor(acc, off, 64);
    const float inv = 1.0f / sqrtf(acc / (float)a.head_dim + a.eps);
    float wv0[CV], wv1[CV];
    dt_decode_raw<DT, CV>(w0, wv0);
    dt_decode_raw<DT, CV>(w1, wv1);
    if (rot) {
#pragma unroll
      for (int e = 0; e < CV; ++e) {
        f0[e] = f0[e] * inv * wv0[e];
        f1[e] = f1[e] * inv * wv1[e];
      }
    }
  }
  if (!live) return;
  if (rot) {
    float cv[CV], sv[CV];
    dt_decode_raw<CT, CV>(c, cv);
    dt_decode_raw<CT, CV>(s, sv);
#pragma unroll
    for (int e = 0; e < CV; ++e) {
      const float y0 = f0[e], y1 = f1[e];
      f0[e] = y0 * cv[e] - y1 * sv[e];
      f1[e] = y1 * cv[e] + y0 * sv[e];
    }
  }
  void *dst;
  int64_t at;
  if (hh < a.n_head) {
    dst = a.q_out;
    at = (int64_t)t * a.q_out_stride + (int64_t)hh * a.head_dim;
  } else {
    const int g = (hh - a.n_head) % a.n_kv_heads;
    dst = rot ? a.k_cache : a.v_cache;
    at = ((((int64_t)tk.page * a.n_kv_heads + g) << a.page_log2) + (tk.pos & ((1 << a.page_log2) - 1))) * a.head_dim;
  }
  dt_store_vec<DT, CV>(dst, at + j, f0);
  dt_store_vec<DT, CV>(dst, at + half + j, f1);
}

namespace {
template <int DT, int CT>
hipError_t launch_append(const PagedAppendArgs &a, hipStream_t st) {
  // Pieces of 8 values; 4 where half a head is no multiple of 8 (72).
  const int half = a.head_dim / 2, cv = half % 8 == 0 ? 8 : 4;
  AppendGeom ag{};
  while ((cv << ag.lpr_log2) < half) ++ag.lpr_log2;
  ag.rows = a.n_tokens * (a.n_head + 2 * a.n_kv_heads);
  const int per_block = 256 >> ag.lpr_log2;
  const dim3 grid((unsigned)((ag.rows + per_block - 1) / per_block));
  if (cv == 8)
    hipLaunchKernelGGL((paged_append_kernel<DT, CT, 8>), grid, dim3(256), 0, st, a, ag);
  else
    hipLaunchKernelGGL((paged_append_kernel<DT, CT, 4>), grid, dim3(256), 0, st, a, ag);
  return hipGetLastError();
}
}  // namespace

hipError_t rk_launch_paged_append(const PagedAppendArgs &a, int dtype, int cs_dtype, hipStream_t st) {
  const bool f32 = cs_dtype == RK_DTYPE_F32;
  if (dtype == RK_DTYPE_F16)
    return f32 ? launch_append<RK_DTYPE_F16, RK_DTYPE_F32>(a, st) : launch_append<RK_DTYPE_F16, RK_DTYPE_F16>(a, st);
  if (dtype == RK_DTYPE_BF16)
    return f32 ? launch_append<RK_DTYPE_BF16, RK_DTYPE_F32>(a, st) : launch_append<RK_DTYPE_BF16, RK_DTYPE_BF16>(a, st);
  return hipErrorInvalidValue;
}
