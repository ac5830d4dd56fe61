// Attention of a batch of sequences: new tokens over the pages of a KV cache, or
// packed sequences over their own keys (items of seq_plan.hpp).
//
// One wave per query row: 64 keys a step, one per lane for the scores, then one
// group of head columns per lane for P·V, with a running maximum and sum.
#include "attn_common.hpp"

namespace {
constexpr int WAVES = 4;

// First value of key `key` of the item's sequence, for kv head g.
template <bool PAGED>
__device__ __forceinline__ int64_t key_at(const SeqAttnArgs &a, const SeqItem &it, int key, int g, int64_t tok_stride) {
  if constexpr (PAGED) {
    const int64_t page = a.table[it.table + (key >> a.page_log2)];
    return (((page * a.n_kv_heads + g) << a.page_log2) + (key & ((1 << a.page_log2) - 1))) * a.head_dim;
  } else {
    return (int64_t)(it.tok0 + key) * tok_stride + (int64_t)g * a.head_dim;
  }
}
}  // namespace

template <int DT, bool PAGED>
__global__ __launch_bounds__(WAVES * 64) void attn_seqs_kernel(SeqAttnArgs a) {
  __shared__ float sq[WAVES][256], sp[WAVES][64];
  const SeqItem it = a.items[blockIdx.x / a.n_kv_heads];
  const int g = blockIdx.x % a.n_kv_heads, G = a.n_head / a.n_kv_heads, D = a.head_dim;
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  for (int r = it.row0 + wave; r < min(it.row0 + SEQ_ROWS, it.rows); r += WAVES) {
    const int q = r / G, h = g * G + r % G, t = it.pos0 + q;
    int lo, hi;
    seq_visible(a, t, it.kv_len, lo, hi);
    for (int d = lane; d < D; d += 64)
      sq[wave][d] = dt_load<DT>(a.q, (int64_t)(it.tok0 + q) * a.q_stride + (int64_t)h * D + d);
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = lo; k0 <= hi; k0 += 64) {
      const int key = k0 + lane;
      float s = -INFINITY;
      if (key <= hi) {
        const int64_t at = key_at<PAGED>(a, it, key, g, a.k_stride);
        s = 0.f;
        for (int d = 0; d < D; d += 8) {
          float kv[8];
          dt_load_vec<DT, 8>(a.k, at + d, kv);
          for (int e = 0; e < 8; ++e) s += kv[e] * sq[wave][d + e];
        }
        s *= a.scale;
        if (a.softcap != 0.f) s = a.softcap * tanhf(s / a.softcap);
        if (a.uniform) s = 0.f;
      }
      float mt = s;
      for (int off = 32; off >= 1; off >>= 1) mt = fmaxf(mt, __shfl_xor(mt, off, 64));
      const float mn = fmaxf(m, mt), mu = mn == -INFINITY ? 0.f : mn;
      const float p = key <= hi ? expf(s - mu) : 0.f, al = expf(m - mu);
      m = mn;
      float lt = p;
      for (int off = 32; off >= 1; off >>= 1) lt += __shfl_xor(lt, off, 64);
      l = l * al + lt;
      sp[wave][lane] = p;
      for (int i = 0; i < 4; ++i) o[i] *= al;
      for (int kk = 0; kk < min(64, hi - k0 + 1); ++kk) {
        const int64_t at = key_at<PAGED>(a, it, k0 + kk, g, a.v_stride);
        for (int i = 0; i < 4; ++i)
          if (lane + 64 * i < D) o[i] += sp[wave][kk] * dt_load<DT>(a.v, at + lane + 64 * i);
      }
    }
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < D)
        dt_store<DT>(a.out, (int64_t)(it.tok0 + q) * a.out_stride + (int64_t)h * D + lane + 64 * i, o[i] / l);
  }
}

hipError_t rk_launch_attention_seqs(const SeqAttnArgs &a, int n_items, bool paged, int dtype, hipStream_t st) {
  const dim3 grid((unsigned)(n_items * a.n_kv_heads)), block(WAVES * 64);
  if (dtype == RK_DTYPE_F16) {
    if (paged) hipLaunchKernelGGL((attn_seqs_kernel<RK_DTYPE_F16, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((attn_seqs_kernel<RK_DTYPE_F16, false>), grid, block, 0, st, a);
  } else if (dtype == RK_DTYPE_BF16) {
    if (paged) hipLaunchKernelGGL((attn_seqs_kernel<RK_DTYPE_BF16, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((attn_seqs_kernel<RK_DTYPE_BF16, false>), grid, block, 0, st, a);
  } else {
    return hipErrorInvalidValue;
  }
  return hipGetLastError();
}
