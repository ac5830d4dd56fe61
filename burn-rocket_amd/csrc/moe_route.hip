// The router of a mixture of experts, and the lists of expert tiles that its choices make, both on the GPU: a routed layer
// needs nothing from the host between its launches and can be captured into a graph.
#include <cfloat>

#include "common.hpp"
#include "kernels.hpp"
#include "moe_tiles.hpp"

// ---------------------------------------------------------------------------
// Router. A wave per token, V consecutive experts a lane. Choices are those of the f64 scores with their bias, or, where
// there is none, of the logits themselves, which order the experts as their scores do: of two experts whose f32 scores are a
// rounding apart the larger is taken, whatever the order of a sum. Equal ones go to the lower id; a NaN ranks with -inf.
//
// What bounds it is the picks, one maximum over the wave each. They go by 32-bit keys that order as the floats do: each lane
// sorts its own, so that a pick is a maximum of the lanes' heads (lane exchanges inside the vector instruction), a ballot, and
// a step of one lane's queue. With a bias the f32 sums decide wherever neighbours in the order are further apart than the
// sums can be off; a token where two are not (about one in four thousand) is done again in f64. 16384 tokens, 256 experts, top 8
// of 4 groups of 8 on MI355X: 18.4 us, 18.7 with a bias of -1e9 on every third expert (52 with a search of all registers per pick and two maxima per group, 95 in f64).
namespace {
constexpr int ROUTE_WAVES = 4;

// Floats to unsigned numbers in the same order, all above 0; -0 as 0, NaN as -inf.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (!(x == x)) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// x of other lanes, inside the vector instruction that uses it (0, which no maximum sees, where there is none): with the
// neighbour, with the neighbouring pair, mirrored in 8 and in 16 lanes (after the two before them: with the other four, the
// other eight); the last lane of a row of 16 to the next row, of the first two rows to the last two.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
constexpr int DPP_1 = 0xB1, DPP_2 = 0x4E, DPP_4 = 0x141, DPP_8 = 0x140, DPP_ROW1 = 0x142, DPP_ROW2 = 0x143;
// The wave's largest key.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = max(x, dpp<DPP_1>(x));
  x = max(x, dpp<DPP_2>(x));
  x = max(x, dpp<DPP_4>(x));
  x = max(x, dpp<DPP_8>(x));
  x = max(x, dpp<DPP_ROW1, 0xa>(x));
  x = max(x, dpp<DPP_ROW2, 0xc>(x));
  return __builtin_amdgcn_readlane(x, 63);
}
// The two largest of 2^n lanes, from the two of each.
__device__ __forceinline__ void join2(uint32_t &a, uint32_t &b, uint32_t oa, uint32_t ob) {
  b = max(min(a, oa), max(b, ob));
  a = max(a, oa);
}
__device__ __forceinline__ void segment_top2(uint32_t &a, uint32_t &b, int lanes) {
  if (lanes > 1) join2(a, b, dpp<DPP_1>(a), dpp<DPP_1>(b));
  if (lanes > 2) join2(a, b, dpp<DPP_2>(a), dpp<DPP_2>(b));
  if (lanes > 4) join2(a, b, dpp<DPP_4>(a), dpp<DPP_4>(b));
  if (lanes > 8) join2(a, b, dpp<DPP_8>(a), dpp<DPP_8>(b));
  if (lanes > 16) join2(a, b, __shfl_xor(a, 16), __shfl_xor(b, 16));
  if (lanes > 32) join2(a, b, __shfl_xor(a, 32), __shfl_xor(b, 32));
}

// A lane's experts in the order they are chosen (key 0: none), by exchanges of neighbours: equal keys keep their order.
template <int V, typename K>
struct Queue {
  K k[V];
  int id[V];
  __device__ __forceinline__ void sort() {
#pragma unroll
    for (int n = V - 1; n > 0; --n)
#pragma unroll
      for (int v = 0; v < n; ++v) {
        const bool swap = k[v + 1] > k[v];
        const K a = k[v], b = k[v + 1];
        const int i = id[v], j = id[v + 1];
        k[v] = swap ? b : a;
        k[v + 1] = swap ? a : b;
        id[v] = swap ? j : i;
        id[v + 1] = swap ? i : j;
      }
  }
  // The ids (below 16: the expert's place in its lane), four bits each, so that a step of the queue moves them at once.
  using Order = std::conditional_t<V <= 8, uint32_t, uint64_t>;
  __device__ __forceinline__ Order order() const {
    Order o = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) o |= (Order)id[v] << (4 * v);
    return o;
  }
  __device__ __forceinline__ void pop(Order &o) {
#pragma unroll
    for (int v = 0; v + 1 < V; ++v) k[v] = k[v + 1];
    k[V - 1] = 0;
    o >>= 4;
  }
};

// The same of f64 numbers, by halves of 64-bit keys.
__device__ __forceinline__ uint64_t order_key(double x) {
  if (!(x == x)) x = -INFINITY;
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | (uint64_t)1 << 63;
}
__device__ __forceinline__ double key_value(uint64_t k) {
  return __longlong_as_double((long long)(k >> 63 ? k & ~((uint64_t)1 << 63) : ~k));
}
__device__ __forceinline__ uint64_t wave_max(uint64_t x) {
  const uint32_t hi = wave_max((uint32_t)(x >> 32));
  const uint32_t lo = wave_max((uint32_t)(x >> 32) == hi ? (uint32_t)x : 0u);
  return (uint64_t)hi << 32 | lo;
}

// Lane j's choice j, with a bias, in f64. Few tokens come here, but the launch waits for them: the same steps as
// below on wider keys, where exchanges of (f64, id) pairs took 25 us.
template <int V>
__device__ __forceinline__ int route_f64(const RouteArgs &g, int64_t t) {
  const int lane = lane_id(), E = g.n_experts;
  double p[V], mx = -INFINITY, sum = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane * V + v;
    p[v] = e < E ? (double)dt_load_any(g.logits, t * E + e, g.dtype) : -INFINITY;
    mx = fmax(mx, p[v]);
  }
  if (g.score == RK_ROUTE_SOFTMAX) {
    for (int d = 1; d < 64; d *= 2) mx = fmax(mx, __shfl_xor(mx, d));
#pragma unroll
    for (int v = 0; v < V; ++v) {
      p[v] = lane * V + v < E ? exp(p[v] - mx) : 0;
      sum += p[v];
    }
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  }
  Queue<V, uint64_t> q;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane * V + v;
    const double s = g.score == RK_ROUTE_SOFTMAX ? p[v] / sum : 1 / (1 + exp(-p[v]));
    q.k[v] = e < E ? order_key(s + (double)g.bias[e]) : 0;
    q.id[v] = v;
  }
  q.sort();
  if (g.top_groups < g.n_groups) {
    uint64_t mine = 0;  // lane i: group i
    for (int i = 0; i < g.n_groups; ++i) {
      uint64_t a = 0, b = 0;  // (sorted: the first two of the group)
#pragma unroll
      for (int v = V - 1; v >= 0; --v)
        if ((lane * V + q.id[v]) / g.group_size == i && q.k[v]) {
          b = a;
          a = q.k[v];
        }
      const uint64_t first = wave_max(a);
      double s = key_value(first);
      if (g.group_size > 1) {
        const int at = __builtin_ctzll(__ballot(a == first));
        s += key_value(wave_max(lane == at ? b : a));
      }
      if (lane == i) mine = order_key(s);
    }
    int rank = 0;
    for (int i = 0; i < g.n_groups; ++i) {
      const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)mine, i);
      rank += o > mine || (o == mine && i < lane);
    }
    const uint64_t kept = __ballot(lane < g.n_groups && rank < g.top_groups);
#pragma unroll
    for (int v = 0; v < V; ++v) q.k[v] = kept >> min((lane * V + q.id[v]) / g.group_size, 63) & 1 ? q.k[v] : 0;
    q.sort();
  }
  int id = 0;
  auto order = q.order();
  for (int j = 0; j < g.top_k; ++j) {
    const uint64_t m = wave_max(q.k[0]);
    const int at = __builtin_ctzll(__ballot(q.k[0] == m));
    const int e = at * V + (__builtin_amdgcn_readlane((int)order, at) & 15);
    if (lane == at) q.pop(order);
    if (lane == j) id = e;
  }
  return id;
}
}  // namespace

template <int V>
__device__ __forceinline__ void route_load(const RouteArgs &g, int64_t t, float (&x)[V]) {
  const int e0 = lane_id() * V, E = g.n_experts;
  constexpr int P = V < 4 ? V : 4;
  auto pieces = [&](auto dt_c) {
    constexpr int DT = decltype(dt_c)::value;
#pragma unroll
    for (int p = 0; p < V; p += P) {
      if (E % P == 0 && e0 + p < E) {
        dt_load_vec<DT, P>(g.logits, t * E + e0 + p, x + p);
      } else {
#pragma unroll
        for (int v = p; v < p + P; ++v) x[v] = e0 + v < E ? dt_load<DT>(g.logits, t * E + e0 + v) : -INFINITY;
      }
    }
  };
  if (g.dtype == RK_DTYPE_F32) pieces(ic<RK_DTYPE_F32>{});
  else if (g.dtype == RK_DTYPE_F16) pieces(ic<RK_DTYPE_F16>{});
  else pieces(ic<RK_DTYPE_BF16>{});
}

template <int V, bool BIAS>
__global__ __launch_bounds__(ROUTE_WAVES * 64) void moe_route_kernel(const RouteArgs g) {
  const int64_t t = (int64_t)blockIdx.x * ROUTE_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= g.s) return;
  const int lane = lane_id(), E = g.n_experts;
  const bool softmax = g.score == RK_ROUTE_SOFTMAX;
  float x[V], bias[V], mx = -INFINITY, sum = 1.f;
  route_load(g, t, x);
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = BIAS && lane * V + v < E ? g.bias[lane * V + v] : 0.f;
  if (softmax) {
#pragma unroll
    for (int v = 0; v < V; ++v) mx = fmaxf(mx, x[v]);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) mx = fmaxf(mx, __shfl_xor(mx, d));
    sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) sum += lane * V + v < E ? expf(x[v] - mx) : 0.f;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  }
  Queue<V, uint32_t> q;
  // With a bias: f32 sums further apart than 2·near·m (groups' sums of two: 4·near·m) are in the order of the exact ones, m the
  // larger magnitude of the compared ones, or 1: a sigmoid's sum is off by 3.9·2^-24·m at most (the reciprocal's and the sum's
  // last bit 1 each, 1 + e^-x 1, e^-x 0.5 and its argument 0.33 times p(1 - p), the largest that |x|·p(1 - p) gets to), a sum of
  // two by 9.8; near is 5 of these. A softmax's also has its sum's error, up to 21 roundings of V and 6 additions, in |p1 - p2|:
  // near is 16. What lies further down is off by more only where it is lower by more, so that neighbours are all to look at,
  // and an expert that a bias of -1e9 closes does not make the others unsure. (-inf is exact: its m is the largest finite number.)
  const float near = softmax ? 0x1p-20f : 0x5p-24f;
  float top = 0.f;
  bool unsure = false;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane * V + v;
    float by = x[v];
    if constexpr (BIAS) {
      const float p = softmax ? __builtin_amdgcn_exp2f((x[v] - mx) * 1.44269504f) * __builtin_amdgcn_rcpf(sum)
                              : __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x[v] * -1.44269504f));
      by = p + bias[v];
      top = fmaxf(top, by < INFINITY ? by : 0.f);
    }
    q.k[v] = e < E ? order_key(by) : 0u;
    q.id[v] = v;
  }
  q.sort();

  // Groups: the score of one is its best choice, or with a bias the sum of its two best; experts of the others are closed.
  if (g.top_groups < g.n_groups) {
    // Groups of 2^shift lanes side by side (-1: other ones).
    const int shift = g.group_shift, lanes = 1 << max(shift, 0), size = g.group_size;
    uint32_t mine = 0;  // lane i: group i
    if (shift >= 0) {
      uint32_t a = q.k[0], b = V > 1 ? q.k[V > 1 ? 1 : 0] : 0u;
      segment_top2(a, b, lanes);
      const uint32_t s = BIAS && g.group_size > 1 ? order_key(key_value(a) + key_value(b)) : a;
      mine = __shfl(s, lane * lanes & 63);
      if (lane >= g.n_groups) mine = 0;
    } else {
      int by = size;
      asm volatile("" : "+s"(by));  // (the divisions stay in this branch)
      for (int i = 0; i < g.n_groups; ++i) {
        uint32_t a = 0, b = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const uint32_t k = (lane * V + q.id[v]) / by == i ? q.k[v] : 0u;
          join2(a, b, k, 0u);
        }
        segment_top2(a, b, 64);
        if (lane == i) mine = BIAS && g.group_size > 1 ? order_key(key_value(a) + key_value(b)) : a;
      }
    }
    // A group's rank: the groups before it.
    int rank = 0;
    for (int i = 0; i < g.n_groups; ++i) {
      const uint32_t o = __builtin_amdgcn_readlane(mine, i);
      rank += o > mine || (o == mine && i < lane);
    }
    const uint64_t kept = __ballot(lane < g.n_groups && rank < g.top_groups);
    if constexpr (BIAS) {
      const int in = __builtin_ctzll(__ballot(lane < g.n_groups && rank == g.top_groups - 1));
      const int out = __builtin_ctzll(__ballot(lane < g.n_groups && rank == g.top_groups));
      const float last = key_value((uint32_t)__builtin_amdgcn_readlane(mine, in)), first = key_value((uint32_t)__builtin_amdgcn_readlane(mine, out));
      // What a sum of two, s, is made of is at most top, and where negative at least s - top, or s: magnitudes of up to
      // max(top, 1) - min(s, 0). (Sums near the largest magnitude may be infinite in f32 alone.)
      const float m = fmaxf(1.f, __uint_as_float(wave_max(__float_as_uint(top)))) + fminf(fmaxf(-first, 0.f), FLT_MAX);  // (top >= 0: ordered as an integer)
      unsure = !(last - first > 4 * near * m) || last < -0x1p126f;
    }
    if (shift >= 0) {
      const bool keep = kept >> (lane >> shift) & 1;
#pragma unroll
      for (int v = 0; v < V; ++v) q.k[v] = keep ? q.k[v] : 0u;
    } else {  // (a lane may have experts of two groups)
      int by = size;
      asm volatile("" : "+s"(by));
#pragma unroll
      for (int v = 0; v < V; ++v) q.k[v] = kept >> min((lane * V + q.id[v]) / by, 63) & 1 ? q.k[v] : 0u;
      q.sort();
    }
  }

  // The top_k: lane j keeps choice j. With a bias one more, to see how far the last one is from it.
  int id = 0;
  uint32_t key = 0;  // lane j: choice j's (none: 0)
  auto order = q.order();
  const int picks = g.top_k + (BIAS && g.top_k < 64 ? 1 : 0);
  for (int j = 0; j < picks; ++j) {
    const uint32_t m = wave_max(q.k[0]);
    if (BIAS && m == 0) break;  // (as many experts as choices)
    const int at = __builtin_ctzll(__ballot(q.k[0] == m));
    const int e = at * V + (__builtin_amdgcn_readlane((int)order, at) & 15);
    if (lane == at) q.pop(order);
    if (lane == j) {
      id = e;
      if constexpr (BIAS) key = m;
    }
  }
  if constexpr (BIAS) {
    // Neighbours in the order: a lane's choice and the next one's.
    const uint32_t behind = g.top_k == 64 ? wave_max(q.k[0]) : 0u, after = __shfl_down(key, 1);
    const uint32_t next = lane < 63 ? after : behind;
    const float mine = key_value(key), other = key_value(next);
    const float m = fminf(fmaxf(fmaxf(1.f, fabsf(mine)), fabsf(other)), FLT_MAX);
    unsure |= __ballot(lane < g.top_k && next != 0 && !(mine - other > 2 * near * m)) != 0;
  }
  if (BIAS && unsure) id = route_f64<V>(g, t);
  // Lane j's weight: the score of its choice's logit.
  float w = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float l = __shfl(x[v], id / V);
    w = v == id % V ? l : w;
  }
  w = lane >= g.top_k ? 0.f : softmax ? expf(w - mx) / sum : 1.0f / (1.0f + expf(-w));
  if (g.norm) {
    float all = w;
    if (g.top_k <= 16) {  // all in one row of lanes
      const auto turned = [&](auto by_c) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(all), decltype(by_c)::value, 0xf, 0xf, false)); };
      all += turned(ic<0x121>{});  // rotations by 1, 2, 4 and 8 lanes
      all += turned(ic<0x122>{});
      all += turned(ic<0x124>{});
      all += turned(ic<0x128>{});
    } else {
#pragma unroll
      for (int d = 1; d < 64; d *= 2) all += __shfl_xor(all, d);
    }
    w = w / (all + 1e-20f);
  }
  if (lane < g.top_k) {
    g.ids[t * g.top_k + lane] = (uint32_t)id;
    g.wts[t * g.top_k + lane] = w * g.scale;
  }
}

hipError_t rk_launch_moe_route(const RouteArgs &args, hipStream_t st) {
  RouteArgs g = args;
  const int v = g.n_experts <= 64 ? 1 : g.n_experts <= 128 ? 2 : g.n_experts <= 256 ? 4 : g.n_experts <= 512 ? 8 : 16;
  g.group_size = g.n_experts / g.n_groups;
  g.group_shift = -1;
  for (int sh = 0; sh <= 6; ++sh)
    if (g.group_size == v << sh) g.group_shift = sh;
#define RK_ROUTE(V) (g.bias ? moe_route_kernel<V, true> : moe_route_kernel<V, false>)
  auto kern = v == 1 ? RK_ROUTE(1) : v == 2 ? RK_ROUTE(2) : v == 4 ? RK_ROUTE(4) : v == 8 ? RK_ROUTE(8) : RK_ROUTE(16);
#undef RK_ROUTE
  hipLaunchKernelGGL(kern, dim3((unsigned)((g.s + ROUTE_WAVES - 1) / ROUTE_WAVES)), dim3(ROUTE_WAVES * 64), 0, st, g);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Lists of a routed batch: the (token, slot) pairs sorted by expert, stably, which is the order that the host's lists have;
// tiles of at most tile_rows rows; each token's rows in ascending expert id. Pairs whose id names no expert form a bucket
// behind the last expert's, whose tiles have expert -1.
//
// Blocks of 1024 pairs. A pair's row is its expert's first row, plus the expert's pairs in earlier blocks, plus those of
// earlier waves of its block, plus those of earlier lanes of its wave. The pairs of other blocks are counted by each block
// itself while there are few, and in a launch of their own that leaves the blocks' counts in memory. No pair waits for
// another block's, and nothing depends on the order of atomics. Bound by the trips to memory one behind the other: 8192 pairs
// over 128 experts on MI355X 8.7 us, 49152 over 64 8.6 and 2.7 for the counts.
namespace {
constexpr int LB = 1024;       // pairs per block
constexpr int LW = LB / 64;
constexpr int COUNT_SELF = 8;  // blocks that count the others' pairs themselves
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

// Where pair j of token t, of expert e, comes among the token's in ascending expert id (the same expert twice: in their order).
__device__ __forceinline__ int place_in_token(const RouteListArgs &g, int64_t t, int e, int j) {
  int at = 0;
  for (int o0 = 0; o0 < g.top_k; o0 += 8) {
    int oe[8];
#pragma unroll
    for (int o = 0; o < 8; ++o) oe[o] = o0 + o < g.top_k ? (int)min(g.ids[t * g.top_k + o0 + o], (uint32_t)g.n_experts) : INT_MAX;
#pragma unroll
    for (int o = 0; o < 8; ++o) at += oe[o] < e || (oe[o] == e && o0 + o < j);
  }
  return at;
}

__global__ __launch_bounds__(LB) void moe_lists_kernel(const RouteListArgs g, int n_blocks) {
  constexpr int ME = RK_ROUTE_MAX_EXPERTS;
  __shared__ int s_all[ME + 1], s_at[ME + 1];   // rows of each expert; those of earlier blocks, then the first row of this one's
  __shared__ uint16_t s_cnt[LW][ME + 1];        // rows of each expert in each wave
  __shared__ uint64_t s_wave[LW];
  const int E = g.n_experts, tid = threadIdx.x, lane = lane_id(), wave = tid >> 6, block = blockIdx.x;
  const bool counted = n_blocks > COUNT_SELF;
  const int64_t i = (int64_t)block * LB + tid;
  const bool in = i < g.rows;
  // Pairs of the other blocks, if they are counted here: on the way while the tables are cleared.
  int other[COUNT_SELF];
#pragma unroll
  for (int b = 0; b < COUNT_SELF; ++b) {
    const int64_t o = (int64_t)b * LB + tid;
    other[b] = !counted && b < n_blocks && o < g.rows ? (int)min(g.ids[o], (uint32_t)E) : -1;
  }
  const int e = in ? (int)min(g.ids[i], (uint32_t)E) : E + 1;
  const int t = (int)(in ? i : 0) / g.top_k;
  const float weight = in && e < E ? g.wts[i] : 0.f;
  const int at = in ? place_in_token(g, t, e, (int)(i - (int64_t)t * g.top_k)) : 0;
  for (int x = tid; x <= E; x += LB) {
    s_all[x] = s_at[x] = 0;
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
  // Rows of each expert in all blocks, and in those before this one.
  if (counted) {
    for (int x = tid; x <= E; x += LB) {
      int all = 0, before = 0;
      const int32_t *c = g.counts + x;
#pragma unroll 8
      for (int b = 0; b < n_blocks; ++b) {
        const int n = c[(int64_t)b * (E + 1)];
        all += n;
        before += b < block ? n : 0;
      }
      s_all[x] = all;
      s_at[x] = before;
    }
  } else if (n_blocks == 1 && block == 0) {
    if (in && rank == 0) atomicAdd(&s_all[e], __popcll(peers));
  } else {
#pragma unroll
    for (int b = 0; b < COUNT_SELF; ++b)
      if (other[b] >= 0) {
        atomicAdd(&s_all[other[b]], 1);
        if (b < block) atomicAdd(&s_at[other[b]], 1);
      }
  }
  __syncthreads();
  const int all = tid < E ? s_all[tid] : 0;
  uint64_t valid;
  const int first = (int)block_exclusive((uint64_t)all, s_wave, &valid);
  if (tid < E) s_at[tid] += first;
  if (tid == 0) s_at[E] += (int)valid;
  __syncthreads();
  if (in) {
    int row = s_at[e] + rank;
    for (int w = 0; w < wave; ++w) row += s_cnt[w][e];
    g.tok[row] = t;
    g.row_w[row] = weight;
    g.slot[(int64_t)t * g.top_k + at] = row;
  }
  if (block < n_blocks) return;

  // Tiles in expert order, and longest first. Thread x makes expert x's.
  const int T = g.tile_rows;
  uint64_t total;
  const uint64_t before = block_exclusive(moe_tile_counts(all, T), s_wave, &total);
  const int n = moe_tile_sum(total);
  if (tid < E)
    moe_tile_places(all, T, before, total, [&](int at, int at_gu, int r, int rows) {
      const MoeTile tile{tid, first + r, rows};
      g.tiles[at] = tile;
      g.tiles_gu[at_gu] = tile;
    });
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
  if (nb > COUNT_SELF) hipLaunchKernelGGL(moe_count_kernel, dim3(nb), dim3(LB), 0, st, g);
  hipLaunchKernelGGL(moe_lists_kernel, dim3(nb + 1), dim3(LB), 0, st, g, nb);
  return hipGetLastError();
}
int rk_moe_lists_blocks(int64_t rows) { return (int)((rows + LB - 1) / LB); }

// Few tokens: no sorting over the batch, one trip to memory instead of four one behind the other (2 us instead of 6).
__global__ __launch_bounds__(256) void moe_pairs_kernel(const RouteListArgs g) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= g.rows) return;
  const int64_t t = i / g.top_k;
  const int e = (int)min(g.ids[i], (uint32_t)g.n_experts), row = (int)(t * g.top_k) + place_in_token(g, t, e, (int)(i - t * g.top_k));
  g.tok[row] = (int32_t)t;
  g.row_w[row] = e < g.n_experts ? g.wts[i] : 0.f;
  g.tiles[row] = g.tiles_gu[row] = MoeTile{e < g.n_experts ? e : -1, row, 1};
}
hipError_t rk_launch_moe_pairs(const RouteListArgs &g, hipStream_t st) {
  hipLaunchKernelGGL(moe_pairs_kernel, dim3((unsigned)((g.rows + 255) / 256)), dim3(256), 0, st, g);
  return hipGetLastError();
}

// The weighted rows of each token to its result, in ascending expert id: y (+)= Σ rows. A thread per eight values; a
// token's rows are asked for four at a time. Bound by the rows' bytes: 49152 fp16 rows of 2048 on MI355X 46 us, 4.4 TB/s.
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
