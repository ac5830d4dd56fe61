// The router of a mixture of experts, and the lists of expert tiles that its choices make, both on the GPU: a routed layer
// needs nothing from the host between its launches and can be captured into a graph.
#include "common.hpp"
#include "kernels.hpp"

// ---------------------------------------------------------------------------
// Router. A wave per token: expert v·64 + lane in register v of the lane. Choices are those of the f64 scores with their
// bias, or, where there is none, of the logits themselves, which order the experts as their scores do: of two experts whose
// f32 scores are a rounding apart the larger is taken, whatever the order of a sum. Equal ones go to the lower id; a NaN
// ranks with -inf.
//
// What bounds it is the picks, one maximum over the wave each: they go by 32-bit keys that order as the floats do (lane
// exchanges inside the vector instruction, then two ballots' worth of scalar work). With a bias the f32 sums decide wherever
// neighbours in the order are further apart than the sums can be off; a token where two are not (about one in a thousand) is
// done again in f64. 16384 tokens, 256 experts, top 8 of 4 groups of 8 on MI355X: ROUTE_US.
namespace {
constexpr int ROUTE_WAVES = 4;

// Floats to unsigned numbers in the same order, all above 0; -0 as 0, NaN as -inf.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (!(x == x)) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false));
}
// The wave's largest key: lanes 1 and 2 apart, mirrored in 8 and 16, then rows into the next ones.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = max_dpp<0xB1>(x);
  x = max_dpp<0x4E>(x);
  x = max_dpp<0x141>(x);
  x = max_dpp<0x140>(x);
  x = max_dpp<0x142>(x);
  x = max_dpp<0x143>(x);
  return __builtin_amdgcn_readlane(x, 63);
}

// Keys of a token's experts (0: not to be chosen), and the picks from them.
template <int V>
struct Keys {
  uint32_t k[V];
  __device__ __forceinline__ uint32_t best() const {
    uint32_t m = k[0];
#pragma unroll
    for (int v = 1; v < V; ++v) m = max(m, k[v]);
    return wave_max(m);
  }
  // The lowest id with the key m.
  __device__ __forceinline__ int find(uint32_t m) const {
    int id = -1;
#pragma unroll
    for (int v = V - 1; v >= 0; --v) {
      const uint64_t has = __ballot(k[v] == m);
      if (has) id = v * 64 + __builtin_ctzll(has);
    }
    return id;
  }
  __device__ __forceinline__ void close(int id) {
#pragma unroll
    for (int v = 0; v < V; ++v) k[v] = v * 64 + lane_id() == id ? 0u : k[v];
  }
};

// f64 form of the choices: (key, id) pairs by lane exchanges.
struct Choice {
  double key;
  int id;  // INT_MAX: none
};
__device__ __forceinline__ bool before(const Choice &a, const Choice &b) { return a.key > b.key || (a.key == b.key && a.id < b.id); }
__device__ __forceinline__ Choice wave_first(Choice c) {
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) {
    const Choice o{__shfl_xor(c.key, d), __shfl_xor(c.id, d)};
    if (before(o, c)) c = o;
  }
  return c;
}

// Ids of lane j's choice j, with a bias, in f64. x: the token's logits (what lies past the last expert is not looked at).
template <int V>
__device__ __forceinline__ int route_f64(const RouteArgs &g, int64_t t) {
  const int lane = lane_id(), E = g.n_experts;
  double key[V], mx = -INFINITY, sum = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 64 + lane;
    key[v] = e < E ? (double)dt_load_any(g.logits, t * E + e, g.dtype) : -INFINITY;
    mx = fmax(mx, key[v]);
  }
  if (g.score == RK_ROUTE_SOFTMAX) {
    for (int d = 1; d < 64; d *= 2) mx = fmax(mx, __shfl_xor(mx, d));
#pragma unroll
    for (int v = 0; v < V; ++v) {
      key[v] = v * 64 + lane < E ? exp(key[v] - mx) : 0;
      sum += key[v];
    }
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  }
  unsigned open = 0;  // experts of the lane that may be chosen
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 64 + lane;
    key[v] = g.score == RK_ROUTE_SOFTMAX ? key[v] / sum : 1 / (1 + exp(-key[v]));
    if (e < E) {
      key[v] += (double)g.bias[e];
      open |= 1u << v;
    }
    if (!(key[v] == key[v])) key[v] = -INFINITY;
  }
  auto best_of = [&](int lo, int hi, unsigned from) {
    Choice c{-INFINITY, INT_MAX};
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = v * 64 + lane;
      const Choice o{key[v], e};
      if ((from >> v & 1) && e >= lo && e < hi && before(o, c)) c = o;
    }
    return wave_first(c);
  };
  auto close = [&](unsigned &mask, int id) {
    if ((id & 63) == lane) mask &= ~(1u << (id >> 6));
  };
  if (g.top_groups < g.n_groups) {
    const int size = E / g.n_groups;
    Choice mine{-INFINITY, INT_MAX};  // lane i: group i
    for (int i = 0; i < g.n_groups; ++i) {
      const Choice a = best_of(i * size, (i + 1) * size, open);
      double s = a.key;
      if (size > 1) {
        unsigned rest = open;
        close(rest, a.id);
        s += best_of(i * size, (i + 1) * size, rest).key;
      }
      if (!(s == s)) s = -INFINITY;  // (two infinities)
      if (lane == i) mine = Choice{s, i};
    }
    uint64_t kept = 0;
    for (int j = 0; j < g.top_groups; ++j) {
      const Choice c = wave_first(mine);
      kept |= (uint64_t)1 << c.id;
      if (lane == c.id) mine = Choice{-INFINITY, INT_MAX};
    }
    unsigned keep = 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if ((open >> v & 1) && (kept >> ((v * 64 + lane) / size) & 1)) keep |= 1u << v;
    open = keep;
  }
  int id = 0;
  for (int j = 0; j < g.top_k; ++j) {
    const Choice c = best_of(0, E, open);
    close(open, c.id);
    if (lane == j) id = c.id;
  }
  return id;
}
}  // namespace

template <int V, bool BIAS>
__global__ __launch_bounds__(ROUTE_WAVES * 64) void moe_route_kernel(const RouteArgs g) {
  const int lane = lane_id();
  const int64_t t = (int64_t)blockIdx.x * ROUTE_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= g.s) return;
  const int E = g.n_experts;
  const bool softmax = g.score == RK_ROUTE_SOFTMAX;
  float x[V], mx = -INFINITY, sum = 1.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 64 + lane;
    x[v] = e < E ? dt_load_any(g.logits, t * E + e, g.dtype) : -INFINITY;
    mx = fmaxf(mx, x[v]);
  }
  if (softmax) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) mx = fmaxf(mx, __shfl_xor(mx, d));
    sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) sum += v * 64 + lane < E ? expf(x[v] - mx) : 0.f;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  }
  auto score = [&](float l) { return softmax ? expf(l - mx) / sum : 1.0f / (1.0f + expf(-l)); };
  Keys<V> keys;
  float most = 1.f;  // the largest finite |score + bias|, at least 1
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 64 + lane;
    float by = x[v];
    if constexpr (BIAS) {
      by = score(x[v]) + (e < E ? g.bias[e] : 0.f);
      if (fabsf(by) < INFINITY) most = fmaxf(most, fabsf(by));
    }
    keys.k[v] = e < E ? order_key(by) : 0u;
  }
  // A f32 sum is off by a few roundings of the score and one of its own: closer ones than this are not told apart.
  float near = 0.f;
  bool unsure = false;
  if constexpr (BIAS) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
    near = most * 0x1p-20f;
  }

  // Groups: the score of one is its best choice, or with a bias the sum of its two best; experts of the others are closed.
  if (g.top_groups < g.n_groups) {
    const int size = E / g.n_groups;
    uint32_t mine = 0;  // lane i: group i
    int group[V];
#pragma unroll
    for (int v = 0; v < V; ++v) group[v] = (v * 64 + lane) / size;
    for (int i = 0; i < g.n_groups; ++i) {
      Keys<V> in;
#pragma unroll
      for (int v = 0; v < V; ++v) in.k[v] = group[v] == i ? keys.k[v] : 0u;
      const uint32_t a = in.best();
      float s = key_value(a);
      if (BIAS && size > 1) {
        in.close(in.find(a));
        s += key_value(in.best());
      }
      if (lane == i) mine = order_key(s);
    }
    uint64_t kept = 0;
    float last = 0.f;
    for (int j = 0; j < g.top_groups + (BIAS ? 1 : 0); ++j) {
      const uint32_t m = wave_max(mine);
      if (BIAS && j == g.top_groups) {
        unsure |= !(last - key_value(m) > 4 * near);
        break;
      }
      const int i = __builtin_ctzll(__ballot(mine == m));
      kept |= (uint64_t)1 << i;
      if (lane == i) mine = 0;
      last = key_value(m);
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (!(kept >> (group[v] & 63) & 1)) keys.k[v] = 0u;
  }

  // The top_k: lane j keeps choice j. With a bias one more, to see how far the last one is from it.
  int id = 0;
  float last = INFINITY;
  for (int j = 0; j < g.top_k + (BIAS ? 1 : 0); ++j) {
    const uint32_t m = keys.best();
    if constexpr (BIAS) {
      if (j > 0 && m != 0) unsure |= !(last - key_value(m) > 2 * near);
      last = key_value(m);
      if (j == g.top_k) break;
    }
    const int i = keys.find(m);
    keys.close(i);
    if (lane == j) id = i;
  }
  if (BIAS && unsure) id = route_f64<V>(g, t);
  // Lane j's logit of its choice.
  float w = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float l = __shfl(x[v], id & 63);
    if (v == id >> 6) w = l;
  }
  w = lane < g.top_k ? score(w) : 0.f;
  if (g.norm) {
    float all = w;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) all += __shfl_xor(all, d);
    w = w / (all + 1e-20f);
  }
  if (lane < g.top_k) {
    g.ids[t * g.top_k + lane] = (uint32_t)id;
    g.wts[t * g.top_k + lane] = w * g.scale;
  }
}

hipError_t rk_launch_moe_route(const RouteArgs &g, hipStream_t st) {
  const int v = (g.n_experts + 63) / 64;
#define RK_ROUTE(V) (g.bias ? moe_route_kernel<V, true> : moe_route_kernel<V, false>)
  auto kern = v <= 1 ? RK_ROUTE(1) : v <= 2 ? RK_ROUTE(2) : v <= 4 ? RK_ROUTE(4) : v <= 8 ? RK_ROUTE(8) : RK_ROUTE(16);
#undef RK_ROUTE
  hipLaunchKernelGGL(kern, dim3((unsigned)((g.s + ROUTE_WAVES - 1) / ROUTE_WAVES)), dim3(ROUTE_WAVES * 64), 0, st, g);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Lists of a routed batch: the (token, slot) pairs sorted by expert, stably, which is the order that the host's lists have;
// tiles of at most tile_rows rows; each token's rows in ascending expert id. Pairs whose id names no expert form a bucket
// behind the last expert's, whose tiles have expert -1.
//
// Blocks of 1024 pairs. A pair's row is its expert's first row, plus the expert's pairs in earlier blocks (from the blocks'
// counts, which a first launch leaves in memory where there are several), plus those of earlier waves of its block, plus
// those of earlier lanes of its wave. No pair waits for another block's, and nothing depends on the order of atomics.
namespace {
constexpr int LB = 1024;       // pairs per block
constexpr int LW = LB / 64;
}  // namespace

__global__ __launch_bounds__(LB) void moe_count_kernel(const RouteListArgs g) {
  __shared__ int cnt[RK_ROUTE_MAX_EXPERTS + 1];
  const int E = g.n_experts;
  for (int e = threadIdx.x; e <= E; e += LB) cnt[e] = 0;
  __syncthreads();
  const int64_t i = (int64_t)blockIdx.x * LB + threadIdx.x;
  if (i < g.rows) atomicAdd(&cnt[min(g.ids[i], (uint32_t)E)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += LB) g.counts[(int64_t)blockIdx.x * (E + 1) + e] = cnt[e];
}

// Exclusive sums of x over the block's threads (fields of a word may be packed: none may carry).
__device__ __forceinline__ uint64_t block_exclusive(uint64_t x, uint64_t *s_wave, uint64_t *total) {
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  uint64_t inc = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t o = __shfl_up(inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 63) s_wave[wave] = inc;
  __syncthreads();
  uint64_t base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < LW; ++w) {
    const uint64_t o = s_wave[w];
    if (w < wave) base += o;
    all += o;
  }
  __syncthreads();
  *total = all;
  return base + inc - x;
}

__global__ __launch_bounds__(LB) void moe_lists_kernel(const RouteListArgs g, int n_blocks) {
  constexpr int ME = RK_ROUTE_MAX_EXPERTS;
  __shared__ int s_all[ME + 1], s_at[ME + 1];   // rows of each expert; the first row of this block's
  __shared__ uint16_t s_cnt[LW][ME + 1];        // rows of each expert in each wave
  __shared__ uint64_t s_wave[LW];
  const int E = g.n_experts, tid = threadIdx.x, lane = lane_id(), wave = tid >> 6;
  const int64_t i = (int64_t)blockIdx.x * LB + tid;
  const bool in = i < g.rows;
  const int e = in ? (int)min(g.ids[i], (uint32_t)E) : E + 1;
  for (int x = tid; x <= E; x += LB) {
    s_all[x] = 0;
#pragma unroll
    for (int w = 0; w < LW; ++w) s_cnt[w][x] = 0;
  }
  __syncthreads();
  // Lanes of the wave with this pair's expert.
  uint64_t peers = ~(uint64_t)0;
  for (int b = 0; (E + 1) >> b != 0; ++b) {
    const uint64_t has = __ballot(e >> b & 1);
    peers &= (e >> b & 1) ? has : ~has;
  }
  const int rank = __popcll(peers & (((uint64_t)1 << lane) - 1));
  if (in && rank == 0) s_cnt[wave][e] = (uint16_t)__popcll(peers);
  if (n_blocks == 1) {
    if (in && rank == 0) atomicAdd(&s_all[e], __popcll(peers));
    __syncthreads();
  }
  // Rows of each expert in all blocks, and in those before this one. (E + 1 may be one more than the threads: the last
  // bucket's count is not needed for the first rows.)
  int all = 0, earlier = 0;
  if (tid < E) {
    if (n_blocks == 1) {
      all = s_all[tid];
    } else {
      for (int b = 0; b < n_blocks; ++b) {
        const int c = g.counts[(int64_t)b * (E + 1) + tid];
        all += c;
        if (b < (int)blockIdx.x) earlier += c;
      }
    }
  }
  uint64_t valid;
  const int first = (int)block_exclusive((uint64_t)all, s_wave, &valid);
  if (tid < E) s_at[tid] = first + earlier;
  if (tid == 0) {
    // The bucket without an expert: what this block and the earlier ones leave over.
    int mine = 0;
    if (n_blocks > 1)
      for (int b = 0; b < (int)blockIdx.x; ++b) mine += g.counts[(int64_t)b * (E + 1) + E];
    s_at[E] = (int)valid + mine;
  }
  __syncthreads();
  if (in) {
    int row = s_at[e] + rank;
    for (int w = 0; w < wave; ++w) row += s_cnt[w][e];
    const int64_t t = i / g.top_k;
    const int j = (int)(i - t * g.top_k);
    g.tok[row] = (int32_t)t;
    g.row_w[row] = e < E ? g.wts[i] : 0.f;
    int at = 0;
    for (int o = 0; o < g.top_k; ++o) {
      const int oe = (int)min(g.ids[t * g.top_k + o], (uint32_t)E);
      if (oe < e || (oe == e && o < j)) ++at;
    }
    g.slot[t * g.top_k + at] = row;
  }
  if (blockIdx.x != 0) return;

  // Tiles in expert order, and longest first: by quarters of tile_rows, in expert order within one. Thread x makes expert
  // x's; four 16-bit counts (quarters 4, 3, 2, 1) share a word of the sums.
  const int T = g.tile_rows, quarter = T / 4;
  auto kinds = [&](int rows) -> uint64_t {
    const int tail = rows % T;
    uint64_t k = (uint64_t)(rows / T);
    if (tail) k += (uint64_t)1 << (16 * (4 - (tail + quarter - 1) / quarter));
    return k;
  };
  uint64_t total;
  const uint64_t mine = kinds(all), base = block_exclusive(mine, s_wave, &total);
  auto field = [](uint64_t x, int f) { return (int)(x >> (16 * f) & 0xffff); };
  auto sum4 = [&](uint64_t x) { return field(x, 0) + field(x, 1) + field(x, 2) + field(x, 3); };
  int start[4];
  for (int f = 0, at = 0; f < 4; ++f) {
    start[f] = at;
    at += field(total, f);
  }
  const int n = sum4(total);
  if (tid < E) {
    int at = sum4(base), full = start[0] + field(base, 0);
    for (int r = 0; r < all; r += T) {
      const int rows = min(T, all - r), f = 4 - (rows + quarter - 1) / quarter;
      const MoeTile tile{tid, first + r, rows};
      g.tiles[at++] = tile;
      // (an expert has any number of whole tiles, and one shorter one at most: whole ones first in their quarter)
      g.tiles_gu[f == 0 ? full++ : start[f] + field(base, f)] = tile;
    }
  }
  // Rows without an expert, and what no tile uses.
  const int left = (int)g.rows - (int)valid, dead = (left + T - 1) / T;
  for (int x = n + tid; x < g.max_tiles; x += LB) {
    const int d = x - n, r = d * T;
    const MoeTile tile = d < dead ? MoeTile{-1, (int)valid + r, min(T, left - r)} : MoeTile{-1, 0, 0};
    g.tiles[x] = tile;
    g.tiles_gu[x] = tile;
  }
  if (tid == 0) *g.n_valid = (int)valid;
}

hipError_t rk_launch_moe_lists(const RouteListArgs &g, hipStream_t st) {
  const int nb = (int)((g.rows + LB - 1) / LB);
  if (nb > 1) hipLaunchKernelGGL(moe_count_kernel, dim3(nb), dim3(LB), 0, st, g);
  hipLaunchKernelGGL(moe_lists_kernel, dim3(nb), dim3(LB), 0, st, g, nb);
  return hipGetLastError();
}
int rk_moe_lists_blocks(int64_t rows) { return (int)((rows + LB - 1) / LB); }

// The weighted rows of each token to its result, in ascending expert id: y (+)= Σ rows. A thread per eight values; a
// token's rows are asked for four at a time. Bound by the rows' bytes.
template <int DT, bool SCALED>
__global__ __launch_bounds__(256) void moe_combine_kernel(const CombineArgs g) {
  constexpr int V = 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = g.n / V;
  if (i >= g.s * per) return;
  const int64_t t = i / per;
  const int c = (int)(i - t * per) * V, groups = SCALED ? (g.n + g.group - 1) / g.group : 0, at = SCALED ? c / g.group : 0;
  float acc[V];
  if (g.accumulate) {
    if constexpr (DT == RK_DTYPE_F32) {
      dt_load_vec<DT, 4>(g.y, t * g.n + c, acc);
      dt_load_vec<DT, 4>(g.y, t * g.n + c + 4, acc + 4);
    } else {
      dt_load_vec<DT, V>(g.y, t * g.n + c, acc);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
  }
  const int valid = g.n_valid ? *g.n_valid : INT_MAX;
  const int32_t *slot = g.slot + t * g.top_k;
  constexpr int U = 4;
  for (int j0 = 0; j0 < g.top_k; j0 += U) {
    float v[U][V], s[U];
    bool has[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = j0 + u < g.top_k ? slot[j0 + u] : INT_MAX;
      has[u] = r < valid && j0 + u < g.top_k;
      const int64_t row = has[u] ? r : 0;
      if constexpr (SCALED) {
        dt_load_vec<RK_DTYPE_F16, V>(g.rows, row * g.n + c, v[u]);
        s[u] = g.scales[row * groups + at];
      } else {
        dt_load_vec<RK_DTYPE_F32, 4>(g.rows, row * g.n + c, v[u]);
        dt_load_vec<RK_DTYPE_F32, 4>(g.rows, row * g.n + c + 4, v[u] + 4);
        s[u] = 1.f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (has[u])
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += v[u][e] * s[u];  // (powers of two: the products are exact)
  }
  if constexpr (DT == RK_DTYPE_F32) {
    dt_store_vec<DT, 4>(g.y, t * g.n + c, acc);
    dt_store_vec<DT, 4>(g.y, t * g.n + c + 4, acc + 4);
  } else {
    dt_store_vec<DT, V>(g.y, t * g.n + c, acc);
  }
}
hipError_t rk_launch_moe_combine(const CombineArgs &g, int dtype, hipStream_t st) {
  const unsigned grid = (unsigned)((g.s * (g.n / 8) + 255) / 256);
#define RK_COMBINE(DT) (g.scales ? moe_combine_kernel<DT, true> : moe_combine_kernel<DT, false>)
  auto kern = dtype == RK_DTYPE_F32 ? RK_COMBINE(RK_DTYPE_F32) : dtype == RK_DTYPE_F16 ? RK_COMBINE(RK_DTYPE_F16) : RK_COMBINE(RK_DTYPE_BF16);
#undef RK_COMBINE
  hipLaunchKernelGGL(kern, dim3(grid), dim3(256), 0, st, g);
  return hipGetLastError();
}
