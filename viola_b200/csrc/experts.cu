// Expert routing around the grouped (expert) linear: which experts a token goes to, in which order the expert GEMM
// sees the rows, and the way back.
//
//   vb_route_forward / _backward    top-k router: softmax weights, per-expert counts, balance loss and z loss
//   vb_expert_plan                  stable counting sort of the choices: row ranges of the experts, row of every choice
//   vb_expert_dispatch              token rows -> rows sorted by expert
//   vb_expert_combine / _backward   rows sorted by expert -> weighted sum per token (unit weights: dispatch's gradient)
//
// No reduction uses floating-point atomics: sums are parked per block and added in a fixed order by a second launch,
// so results repeat bit for bit, and no workspace needs a particular content before the call.
#include <climits>

#include "api.h"
#include "common/numerics.cuh"

namespace vb {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kMaxExperts = 1024, kMaxTopK = 32;

template <int BYTES> struct Word;
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<16> { using type = uint4; };

template <typename T> __device__ __forceinline__ float to_float(T v) { return (float)v; }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v) { return (T)v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }

// ---- router ---------------------------------------------------------------------------------------------------
// A token is served by G lanes (G = 32, or the next power of two of the expert count below that); lane `sub` of the
// group owns the experts sub * V .. sub * V + V - 1.
template <typename T, int G, int V>
__device__ __forceinline__ void load_values(const T* row, int sub, int experts, bool wide, float (&v)[V]) {
  constexpr int kBytes = V * (int)sizeof(T) >= 16 ? 16 : V * (int)sizeof(T);
  using W = typename Word<kBytes>::type;
  constexpr int kPer = kBytes / (int)sizeof(T);
  if (wide) {
#pragma unroll
    for (int w = 0; w < V / kPer; ++w) {
      const W raw = *reinterpret_cast<const W*>(row + sub * V + w * kPer);
      const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[w * kPer + i] = to_float(t[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = sub * V + i < experts ? to_float(row[sub * V + i]) : -INFINITY;
  }
}
template <typename T, int G, int V>
__device__ __forceinline__ void store_values(T* row, int sub, int experts, bool wide, const float (&v)[V]) {
  constexpr int kBytes = V * (int)sizeof(T) >= 16 ? 16 : V * (int)sizeof(T);
  using W = typename Word<kBytes>::type;
  constexpr int kPer = kBytes / (int)sizeof(T);
  if (wide) {
#pragma unroll
    for (int w = 0; w < V / kPer; ++w) {
      W raw;
      T* t = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int i = 0; i < kPer; ++i) t[i] = from_float<T>(v[w * kPer + i]);
      *reinterpret_cast<W*>(row + sub * V + w * kPer) = raw;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (sub * V + i < experts) row[sub * V + i] = from_float<T>(v[i]);
  }
}

template <int G> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
template <int G> __device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

// Unsigned integers in the order of the keys: -inf is 0 (never chosen), NaN the largest (as a descending sort has it).
__device__ __forceinline__ unsigned ordered(float key) {
  if (key != key) return 0xffffffffu;
  if (key == -INFINITY) return 0u;
  const unsigned bits = __float_as_uint(key + 0.0f);       // -0 + 0 = +0: the two zeros tie
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// softmax of a row: p[i], and its log-sum-exp
template <int G, int V>
__device__ __forceinline__ float group_softmax(const float (&l)[V], float (&p)[V], float& top, float& total) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < V; ++i) m = fmaxf(m, l[i]);
  top = group_max<G>(m);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    p[i] = expf(l[i] - top);
    s += p[i];
  }
  total = group_sum<G>(s);
  const float inverse = 1.f / total;
#pragma unroll
  for (int i = 0; i < V; ++i) p[i] *= inverse;
  return top + logf(total);
}

struct RouteArgs {
  const void* logits;
  long long stride;            // elements
  int tokens, experts, top_k, normalize, wide;
  const float* bias;
  const uint8_t* mask;
  float* weights;
  int* indices;
  int* counts;
  float* balance;
  float* z;
  float* inverse;              // {1 / tokens, 1 / choices}, both at least 1 before the reciprocal
  float* partial;              // [blocks][2 * experts + 2]: sums of p, counts, sum of lse^2, tokens
};

// balance = E * sum_e (counts_e / choices) * (sum_t p_te / tokens) from per-expert totals in shared memory
__device__ __forceinline__ void route_finish(const RouteArgs& a, const float* p_sum, const int* count, float z, int tokens) {
  __shared__ float dot_part[32];
  __shared__ int sum_part[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  float dot = 0.f;
  int sum = 0;
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
    dot = fmaf((float)count[e], p_sum[e], dot);
    sum += count[e];
    a.counts[e] = count[e];
  }
  dot = group_sum<32>(dot);
  sum = __reduce_add_sync(kFull, sum);
  if (lane == 0) {
    dot_part[warp] = dot;
    sum_part[warp] = sum;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    dot = 0.f;
    sum = 0;
    for (int w = 0; w < warps; ++w) {
      dot += dot_part[w];
      sum += sum_part[w];
    }
    const float per_token = 1.f / (float)max(tokens, 1), per_choice = 1.f / (float)max(sum, 1);
    *a.balance = (float)a.experts * dot * per_token * per_choice;
    *a.z = z * per_token;
    a.inverse[0] = per_token;
    a.inverse[1] = per_choice;
  }
}

template <typename T, int G, int V>
__global__ void __launch_bounds__(256)
route_forward_kernel(const RouteArgs a) {
  extern __shared__ float shared[];             // [8][experts] sums of p, [experts] counts
  __shared__ float z_part[8];
  __shared__ int n_part[8];
  constexpr int kTokens = 32 / G;               // tokens a warp serves at a time
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane & (G - 1), base = lane - sub;
  int* count = reinterpret_cast<int*>(shared + 8 * a.experts);
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) count[e] = 0;
  __syncthreads();

  float bias[V], p_sum[V], z_sum = 0.f;
  int live_tokens = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias != nullptr && sub * V + i < a.experts ? a.bias[sub * V + i] : 0.f;
    p_sum[i] = 0.f;
  }
  for (long long first = (long long)(blockIdx.x * 8 + warp) * kTokens; first < a.tokens;
       first += (long long)gridDim.x * 8 * kTokens) {
    const long long token = first + lane / G;
    const bool inside = token < a.tokens, live = inside && (a.mask == nullptr || a.mask[token] != 0);
    float l[V], p[V], top, total;
    unsigned key[V];
    if (live) {
      load_values<T, G, V>(reinterpret_cast<const T*>(a.logits) + token * a.stride, sub, a.experts, a.wide, l);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) l[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = sub * V + i < a.experts ? ordered(l[i] + bias[i]) : 0u;
    const float lse = group_softmax<G, V>(l, p, top, total);

    int my_index = -1;
    float my_logit = -INFINITY;
    for (int j = 0; j < a.top_k; ++j) {
      unsigned best = 0u;
      int at = INT_MAX;
      float logit = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (key[i] > best) {                    // strictly: the lowest index of equal keys stays
          best = key[i];
          at = sub * V + i;
          logit = l[i];
        }
      }
      int index;
      if constexpr (G == 32) {
        const unsigned most = __reduce_max_sync(kFull, best);
        index = most == 0u ? -1 : (int)__reduce_min_sync(kFull, best == most ? (unsigned)at : (unsigned)INT_MAX);
      } else {
        unsigned most = best;
        index = at;
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) {
          const unsigned other = __shfl_xor_sync(kFull, most, o);
          const int other_at = __shfl_xor_sync(kFull, index, o);
          if (other > most || (other == most && other_at < index)) {
            most = other;
            index = other_at;
          }
        }
        if (most == 0u) index = -1;
      }
      const float chosen = __shfl_sync(kFull, logit, base + max(index, 0) / V);
      if (index >= 0 && sub == j) {
        my_index = index;
        my_logit = chosen;
      }
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (sub * V + i == index) key[i] = 0u;
    }

    const bool counted = __shfl_sync(kFull, my_index, base) >= 0;
    float weight;
    if (a.normalize) {                          // softmax over the chosen logits = p / (sum of the chosen p)
      const float most = group_max<G>(my_logit);
      const float e = my_index >= 0 ? expf(my_logit - most) : 0.f;
      weight = e / group_sum<G>(e);
    } else {
      weight = expf(my_logit - top) / total;
    }
    if (inside && sub < a.top_k) {
      a.indices[token * a.top_k + sub] = my_index;
      a.weights[token * a.top_k + sub] = my_index >= 0 ? weight : 0.f;
      if (my_index >= 0) atomicAdd(&count[my_index], 1);
    }
    if (counted) {
#pragma unroll
      for (int i = 0; i < V; ++i) p_sum[i] += p[i];
      if (sub == 0) {
        z_sum = fmaf(lse, lse, z_sum);
        ++live_tokens;
      }
    }
  }

#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int o = G; o < 32; o <<= 1) p_sum[i] += __shfl_xor_sync(kFull, p_sum[i], o);
    if (lane < G && sub * V + i < a.experts) shared[warp * a.experts + sub * V + i] = p_sum[i];
  }
  z_sum = group_sum<32>(z_sum);
  live_tokens = __reduce_add_sync(kFull, live_tokens);
  if (lane == 0) {
    z_part[warp] = z_sum;
    n_part[warp] = live_tokens;
  }
  __syncthreads();
  float z = 0.f;
  int n = 0;
  for (int w = 0; w < 8; ++w) {
    z += z_part[w];
    n += n_part[w];
  }
  float* mine = a.partial + (long long)blockIdx.x * (2 * a.experts + 2);
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
    float total = 0.f;
    for (int w = 0; w < 8; ++w) total += shared[w * a.experts + e];
    if (gridDim.x > 1) {
      mine[e] = total;
      mine[a.experts + e] = __int_as_float(count[e]);
    } else {
      shared[e] = total;                        // column e is read and written by this thread alone
    }
  }
  if (gridDim.x > 1) {
    if (threadIdx.x == 0) {
      mine[2 * a.experts] = z;
      mine[2 * a.experts + 1] = __int_as_float(n);
    }
    return;
  }
  __syncthreads();
  route_finish(a, shared, count, z, n);
}

// Adds the blocks' sums in block order and derives the losses: 1024 threads, `experts` rounded up to a power of two
// columns x as many interleaved row groups as fit.
__global__ void __launch_bounds__(1024)
route_finish_kernel(const RouteArgs a, int blocks, int columns) {
  extern __shared__ float shared[];             // [groups][columns] sums, [groups][columns] counts
  const int groups = 1024 / columns, column = threadIdx.x % columns, group = threadIdx.x / columns;
  int* counts = reinterpret_cast<int*>(shared + 1024);
  const int pitch = 2 * a.experts + 2;
  float p = 0.f;
  int c = 0;
  if (column < a.experts) {
    for (int b = group; b < blocks; b += groups) {
      p += a.partial[(long long)b * pitch + column];
      c += __float_as_int(a.partial[(long long)b * pitch + a.experts + column]);
    }
  }
  shared[group * columns + column] = p;
  counts[group * columns + column] = c;
  float z = 0.f;
  int n = 0;
  if (threadIdx.x < 32) {
    for (int b = threadIdx.x; b < blocks; b += 32) {
      z += a.partial[(long long)b * pitch + 2 * a.experts];
      n += __float_as_int(a.partial[(long long)b * pitch + 2 * a.experts + 1]);
    }
    z = group_sum<32>(z);
    n = __reduce_add_sync(kFull, n);
  }
  __syncthreads();
  if (group == 0) {
    for (int g = 1; g < groups; ++g) {
      p += shared[g * columns + column];
      c += counts[g * columns + column];
    }
    shared[column] = p;
    counts[column] = c;
  }
  __syncthreads();
  route_finish(a, shared, counts, z, n);
}

struct RouteBackwardArgs {
  const void* logits;
  long long stride;
  int tokens, experts, top_k, normalize, wide;
  const float* weights;
  const int* indices;
  const int* counts;
  const float* inverse;
  const float* dweights;       // optional [tokens, top_k]
  const float* dbalance;       // optional scalars
  const float* dz;
  void* dlogits;               // contiguous [tokens, experts]
};

// With S the chosen experts, w their weights and g the gradient of w, f_e = counts_e / choices:
//   normalised:  dl_e = [e in S] w_e (g_e - sum_S w g)          else:  dl_e = p_e ([e in S] g_e - sum_S p g)
//   balance:     dl_e += db * E / tokens * p_e (f_e - sum_e' p_e' f_e')
//   z:           dl_e += dz * 2 / tokens * lse * p_e
// The softmax is formed again from the logits: reading them costs what reading a saved p would.
template <typename T, int G, int V>
__global__ void __launch_bounds__(256)
route_backward_kernel(const RouteBackwardArgs a) {
  constexpr int kTokens = 32 / G;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane & (G - 1), base = lane - sub;
  const float per_token = a.inverse[0], per_choice = a.inverse[1];
  const float cb = a.dbalance != nullptr ? *a.dbalance * (float)a.experts * per_token : 0.f;
  const float cz = a.dz != nullptr ? *a.dz * 2.f * per_token : 0.f;
  float f[V];
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = sub * V + i < a.experts ? (float)a.counts[sub * V + i] * per_choice : 0.f;
  for (long long first = (long long)(blockIdx.x * 8 + warp) * kTokens; first < a.tokens;
       first += (long long)gridDim.x * 8 * kTokens) {
    const long long token = first + lane / G;
    const bool inside = token < a.tokens;
    int index = -1;
    float w = 0.f, g = 0.f;
    if (inside && sub < a.top_k) {
      index = a.indices[token * a.top_k + sub];
      w = a.weights[token * a.top_k + sub];
      if (a.dweights != nullptr) g = a.dweights[token * a.top_k + sub];
      if (index < 0) w = g = 0.f;
    }
    const bool counted = __shfl_sync(kFull, index, base) >= 0;
    float l[V], p[V], top, total;
    if (counted) {
      load_values<T, G, V>(reinterpret_cast<const T*>(a.logits) + token * a.stride, sub, a.experts, a.wide, l);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) l[i] = -INFINITY;
    }
    const float lse = group_softmax<G, V>(l, p, top, total);
    float pf = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) pf = fmaf(p[i], f[i], pf);
    pf = group_sum<G>(pf);
    const float dot = group_sum<G>(w * g);
    const float common = cz * lse - (a.normalize ? 0.f : dot);
    const float own = w * (a.normalize ? g - dot : g);
    float grad[V];
#pragma unroll
    for (int i = 0; i < V; ++i) grad[i] = p[i] * fmaf(cb, f[i] - pf, common);
    for (int j = 0; j < a.top_k; ++j) {
      const int at = __shfl_sync(kFull, index, base + j);
      const float add = __shfl_sync(kFull, own, base + j);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (sub * V + i == at) grad[i] += add;
    }
    if (inside) {
      if (!counted) {
#pragma unroll
        for (int i = 0; i < V; ++i) grad[i] = 0.f;
      }
      store_values<T, G, V>(reinterpret_cast<T*>(a.dlogits) + token * a.experts, sub, a.experts, a.wide, grad);
    }
  }
}

// ---- plan: stable counting sort of the choices -------------------------------------------------------------------
// Every block owns `chunk` consecutive choices, every warp of it a consecutive eighth.  A block's first row for an
// expert is what earlier experts hold altogether plus what earlier blocks hold of this one.
__device__ __forceinline__ int read_choice(const void* indices, int is_long, long long i, int experts) {
  const long long e = is_long ? reinterpret_cast<const long long*>(indices)[i] : (long long)reinterpret_cast<const int*>(indices)[i];
  return e >= 0 && e < experts ? (int)e : -1;
}

__global__ void __launch_bounds__(256)
plan_count_kernel(const void* __restrict__ indices, int is_long, int n, int experts, int chunk, int* __restrict__ histogram) {
  extern __shared__ int plan_shared[];
  for (int e = threadIdx.x; e < experts; e += blockDim.x) plan_shared[e] = 0;
  __syncthreads();
  const long long first = (long long)blockIdx.x * chunk, last = min(first + chunk, (long long)n);
  for (long long i = first + threadIdx.x; i < last; i += blockDim.x) {
    const int e = read_choice(indices, is_long, i, experts);
    if (e >= 0) atomicAdd(&plan_shared[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += blockDim.x) histogram[(long long)blockIdx.x * experts + e] = plan_shared[e];
}

__global__ void __launch_bounds__(256)
plan_place_kernel(const void* __restrict__ indices, int is_long, int n, int experts, int chunk,
                  const int* __restrict__ histogram, int* __restrict__ offsets, int* __restrict__ positions) {
  extern __shared__ int plan_shared[];               // [8][experts] next row of every warp, [experts + 1] first row of every expert
  __shared__ int scan_part[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int* first_row = plan_shared + 8 * experts;
  int* next = plan_shared + warp * experts;
  for (int i = threadIdx.x; i < 8 * experts; i += blockDim.x) plan_shared[i] = 0;
  __syncthreads();
  const long long block_first = (long long)blockIdx.x * chunk, block_last = min(block_first + chunk, (long long)n);
  const long long first = block_first + (long long)warp * (chunk / 8), last = min(first + chunk / 8, block_last);
  for (long long i = first + lane; i < last; i += 32) {
    const int e = read_choice(indices, is_long, i, experts);
    if (e >= 0) atomicAdd(&next[e], 1);
  }
  __syncthreads();
  // totals of all blocks, and of the blocks before this one; a thread owns the consecutive experts 4 t .. 4 t + 3
  int total[4], before[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = threadIdx.x * 4 + i;
    total[i] = before[i] = 0;
    if (e < experts) {
      if (histogram != nullptr) {
        for (int b = 0; b < (int)gridDim.x; ++b) {
          const int c = histogram[(long long)b * experts + e];
          total[i] += c;
          if (b < (int)blockIdx.x) before[i] += c;
        }
      } else {
        for (int w = 0; w < 8; ++w) total[i] += plan_shared[w * experts + e];
      }
    }
    sum += total[i];
  }
  int scan = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int other = __shfl_up_sync(kFull, scan, o);
    if (lane >= o) scan += other;
  }
  if (lane == 31) scan_part[warp] = scan;
  __syncthreads();
  int start = scan - sum;
  for (int w = 0; w < warp; ++w) start += scan_part[w];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = threadIdx.x * 4 + i;
    if (e < experts) {
      first_row[e] = start;
      int row = start + before[i];
      for (int w = 0; w < 8; ++w) {              // turn the warps' counts into their first rows
        const int c = plan_shared[w * experts + e];
        plan_shared[w * experts + e] = row;
        row += c;
      }
      start += total[i];
      if (e == experts - 1) first_row[experts] = start;
    }
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= experts; e += blockDim.x) offsets[e] = first_row[e];
  for (long long i = first; i < last; i += 32) {
    const bool inside = i + lane < last;
    const int e = inside ? read_choice(indices, is_long, i + lane, experts) : -1;
    const unsigned peers = __match_any_sync(kFull, e);
    const int rank = __popc(peers & ((1u << lane) - 1u));
    if (inside) positions[i + lane] = e >= 0 ? next[e] + rank : -1;
    __syncwarp();
    if (e >= 0 && rank == 0) next[e] += __popc(peers);
    __syncwarp();
  }
}

// ---- rows to experts and back -----------------------------------------------------------------------------------
// rows behind the last expert's hold zeros, so that whatever reads the whole buffer (an amax) finds nothing of its own
template <typename W>
__device__ __forceinline__ void clear_tail(W* rows, long long words, long long first, long long last) {
  const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long r = first + (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); r < last; r += warps)
    for (long long c = threadIdx.x & 31; c < words; c += 32) rows[r * words + c] = W{};
}

// One warp per (token, segment of 32 * U words): the token's words are read once and stored top_k times.
template <typename W, int U>
__global__ void __launch_bounds__(256)
dispatch_kernel(const W* __restrict__ x, long long x_words, int words, int segments, int tokens, int top_k,
                const int* __restrict__ positions, const int* __restrict__ offsets, int experts, W* __restrict__ rows) {
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * (blockDim.x >> 5), items = (long long)tokens * segments;
  const long long capacity = (long long)tokens * top_k;
  for (long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); item < items; item += warps) {
    const long long token = item / segments;
    const int first = (int)(item - token * segments) * 32 * U + lane;
    W v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + 32 * u < words) v[u] = x[token * x_words + first + 32 * u];
    for (int j = 0; j < top_k; ++j) {
      const int row = positions[token * top_k + j];
      if (row < 0 || row >= capacity) continue;
      W* to = rows + (long long)row * words;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (first + 32 * u < words) to[first + 32 * u] = v[u];
    }
  }
  clear_tail(rows, words, min(max((long long)offsets[experts], 0LL), capacity), capacity);
}

template <typename T, int N> struct Pack {       // N values of T moved as one word
  using W = typename Word<N * (int)sizeof(T) >= 16 ? 16 : N * (int)sizeof(T)>::type;
  static constexpr int kWords = N * (int)sizeof(T) / (int)sizeof(W);
  W raw[kWords];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) raw[i] = reinterpret_cast<const W*>(p)[i];
  }
  __device__ __forceinline__ void get(float (&v)[N]) const {
    const T* t = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_float(t[i]);
  }
  __device__ __forceinline__ static void store(T* p, const float (&v)[N]) {
    W raw[kWords];
    T* t = reinterpret_cast<T*>(raw);
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = from_float<T>(v[i]);
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<W*>(p)[i] = raw[i];
  }
};

// out[t] = sum_j weights[t, j] * rows[positions[t, j]], added in fp32 in the order of j; weights null: all one
template <typename T, int N, int U>
__global__ void __launch_bounds__(256)
combine_kernel(const T* __restrict__ rows, int width, int segments, int tokens, int top_k, const int* __restrict__ positions,
               const void* __restrict__ weights, int weight_dtype, T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * (blockDim.x >> 5), items = (long long)tokens * segments;
  const long long capacity = (long long)tokens * top_k;
  for (long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); item < items; item += warps) {
    const long long token = item / segments;
    const int first = ((int)(item - token * segments) * 32 * U + lane) * N;
    float sum[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) sum[u][i] = 0.f;
    for (int j = 0; j < top_k; ++j) {
      const int row = positions[token * top_k + j];
      if (row < 0 || row >= capacity) continue;
      const float w = weights != nullptr ? load_as_float(weights, token * top_k + j, weight_dtype) : 1.f;
      Pack<T, N> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (first + 32 * u * N < width) v[u].load(rows + (long long)row * width + first + 32 * u * N);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[N];
        if (first + 32 * u * N < width) {
          v[u].get(f);
#pragma unroll
          for (int i = 0; i < N; ++i) sum[u][i] = fmaf(w, f[i], sum[u][i]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + 32 * u * N < width) Pack<T, N>::store(out + token * width + first + 32 * u * N, sum[u]);
  }
}

// drows[positions[t, j]] = weights[t, j] * dout[t],  dweights[t, j] = <dout[t], rows[positions[t, j]]>
// A token is served by `team` warps of a block (1, 2, 4 or 8), so that its row of dout is read once for rows of up to
// team * 32 * U packs and the dot products end in the block.
template <typename T, int N, int U>
__global__ void __launch_bounds__(256)
combine_backward_kernel(const T* __restrict__ dout, const T* __restrict__ rows, int width, int tokens, int top_k, int team,
                        const int* __restrict__ positions, const int* __restrict__ offsets, int experts,
                        const void* __restrict__ weights, int weight_dtype, T* __restrict__ drows, void* __restrict__ dweights) {
  __shared__ float part[8][kMaxTopK];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per_block = 8 / team, member = warp % team;
  const long long capacity = (long long)tokens * top_k;
  for (long long base = (long long)blockIdx.x * per_block; base < tokens; base += (long long)gridDim.x * per_block) {
    const long long token = base + warp / team;
    if (token < tokens) {
      for (int j = 0; j < top_k; ++j) {
        const int row = positions[token * top_k + j];
        const bool placed = row >= 0 && row < capacity;
        const float w = placed ? load_as_float(weights, token * top_k + j, weight_dtype) : 0.f;
        float dot = 0.f;
        if (placed) {
          for (int first = (member * 32 * U + lane) * N; first < width; first += team * 32 * U * N) {
            Pack<T, N> g[U], v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int c = first + 32 * u * N;
              if (c < width) {
                v[u].load(rows + (long long)row * width + c);
                g[u].load(dout + token * width + c);
              }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int c = first + 32 * u * N;
              if (c < width) {
                float gf[N], vf[N];
                g[u].get(gf);
                v[u].get(vf);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                  dot = fmaf(gf[i], vf[i], dot);
                  gf[i] *= w;
                }
                if (drows != nullptr) Pack<T, N>::store(drows + (long long)row * width + c, gf);
              }
            }
          }
        }
        dot = group_sum<32>(dot);
        if (lane == 0) part[warp][j] = dot;
      }
    }
    if (team > 1) __syncthreads(); else __syncwarp();
    if (token < tokens && member == 0 && lane < top_k && dweights != nullptr) {
      float dot = 0.f;
      for (int m = 0; m < team; ++m) dot += part[warp + m][lane];
      store_from_float(dweights, token * top_k + lane, weight_dtype, dot);
    }
    if (team > 1) __syncthreads(); else __syncwarp();
  }
  if (drows != nullptr) {
    using W = typename Pack<T, N>::W;
    clear_tail(reinterpret_cast<W*>(drows), (long long)width * (int)sizeof(T) / (int)sizeof(W),
               min(max((long long)offsets[experts], 0LL), capacity), capacity);
  }
}

}  // namespace vb

using namespace vb;

static bool aligned_to(const void* p, long long bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// lanes per token and experts per lane
#define VB_ROUTE_SWITCH(experts, ...)                                            \
  if ((experts) <= 4) { constexpr int G = 4, V = 1; __VA_ARGS__; }               \
  else if ((experts) <= 8) { constexpr int G = 8, V = 1; __VA_ARGS__; }          \
  else if ((experts) <= 16) { constexpr int G = 16, V = 1; __VA_ARGS__; }        \
  else if ((experts) <= 32) { constexpr int G = 32, V = 1; __VA_ARGS__; }        \
  else if ((experts) <= 64) { constexpr int G = 32, V = 2; __VA_ARGS__; }        \
  else if ((experts) <= 128) { constexpr int G = 32, V = 4; __VA_ARGS__; }       \
  else if ((experts) <= 256) { constexpr int G = 32, V = 8; __VA_ARGS__; }       \
  else if ((experts) <= 512) { constexpr int G = 32, V = 16; __VA_ARGS__; }      \
  else { constexpr int G = 32, V = 32; __VA_ARGS__; }

#define VB_FLOAT_SWITCH(dtype, ...)                                              \
  if ((dtype) == kF32) { using T = float; __VA_ARGS__; }                         \
  else if ((dtype) == kBF16) { using T = __nv_bfloat16; __VA_ARGS__; }           \
  else { using T = __half; __VA_ARGS__; }

static int route_lanes(int experts) { return experts <= 4 ? 4 : experts <= 8 ? 8 : experts <= 16 ? 16 : 32; }
// blocks of 8 warps
static int route_blocks(int tokens, int experts) {
  const long long per_pass = 8LL * (32 / route_lanes(experts));
  if (tokens <= 4 * per_pass) return 1;
  return (int)std::min<long long>((tokens + per_pass - 1) / per_pass, 148LL * 2);
}
static bool route_wide(const void* p, long long stride, int experts, int size) {
  const int lanes = route_lanes(experts), per_lane = experts / lanes;
  if (experts % lanes || (per_lane & (per_lane - 1))) return false;
  const int bytes = std::min(16, per_lane * size);
  return aligned_to(p, bytes) && stride * size % bytes == 0;
}
static bool route_shape_ok(int tokens, int experts, int top_k, int dtype) {
  return tokens >= 0 && experts >= 1 && experts <= kMaxExperts && top_k >= 1 && top_k <= std::min(experts, kMaxTopK) &&
         dtype >= kF32 && dtype <= kF16;
}

extern "C" long long vb_route_workspace(int tokens, int experts) {
  return tokens < 0 || experts < 1 ? 0 : (long long)route_blocks(tokens, experts) * (2 * experts + 2);
}

extern "C" int vb_route_forward(const void* logits, int dtype, int tokens, int experts, long long stride, const float* bias,
                                const uint8_t* mask, int top_k, int normalize, float* weights, int* indices, int* counts,
                                float* balance, float* z, float* inverse, float* workspace, long long workspace_floats,
                                cudaStream_t stream) {
  if (!route_shape_ok(tokens, experts, top_k, dtype) || workspace == nullptr ||
      workspace_floats < vb_route_workspace(tokens, experts))
    return (int)cudaErrorInvalidValue;
  RouteArgs a{logits, stride, tokens, experts, top_k, normalize, 0, bias, mask, weights, indices, counts, balance, z, inverse,
              workspace};
  a.wide = route_wide(logits, stride, experts, dtype == kF32 ? 4 : 2);
  const int blocks = route_blocks(tokens, experts);
  const size_t smem = (size_t)9 * experts * sizeof(float);
  VB_FLOAT_SWITCH(dtype, VB_ROUTE_SWITCH(experts, (route_forward_kernel<T, G, V><<<blocks, 256, smem, stream>>>(a))));
  if (blocks > 1) {
    int columns = 32;
    while (columns < experts) columns *= 2;
    route_finish_kernel<<<1, 1024, 2048 * sizeof(float), stream>>>(a, blocks, columns);
  }
  return (int)cudaGetLastError();
}

extern "C" int vb_route_backward(const void* logits, int dtype, int tokens, int experts, long long stride, int top_k,
                                 int normalize, const float* weights, const int* indices, const int* counts,
                                 const float* inverse, const float* dweights, const float* dbalance, const float* dz,
                                 void* dlogits, cudaStream_t stream) {
  if (!route_shape_ok(tokens, experts, top_k, dtype)) return (int)cudaErrorInvalidValue;
  if (tokens == 0) return 0;
  RouteBackwardArgs a{logits, stride, tokens, experts, top_k, normalize, 0, weights, indices, counts, inverse, dweights,
                      dbalance, dz, dlogits};
  const int size = dtype == kF32 ? 4 : 2;
  a.wide = route_wide(logits, stride, experts, size) && route_wide(dlogits, experts, experts, size);
  const long long per_pass = 8LL * (32 / route_lanes(experts));
  const int blocks = (int)std::min<long long>((tokens + per_pass - 1) / per_pass, 148LL * 8);
  VB_FLOAT_SWITCH(dtype, VB_ROUTE_SWITCH(experts, (route_backward_kernel<T, G, V><<<blocks, 256, 0, stream>>>(a))));
  return (int)cudaGetLastError();
}

// choices per block: a multiple of 8 warps x 32 lanes; about one block per SM for long lists
static int plan_chunk(int n) {
  const long long per = ((long long)n + 147) / 148;
  return (int)std::max<long long>(4096, (per + 255) / 256 * 256);
}

extern "C" long long vb_expert_plan_workspace(int n, int experts) {
  if (n < 0 || experts < 1) return 0;
  const int chunk = plan_chunk(n);
  return n <= chunk ? 0 : ((long long)n + chunk - 1) / chunk * experts;
}

extern "C" int vb_expert_plan(const void* indices, int is_long, int n, int experts, int* offsets, int* positions,
                              int* workspace, long long workspace_ints, cudaStream_t stream) {
  if (n < 0 || experts < 1 || experts > kMaxExperts || workspace_ints < vb_expert_plan_workspace(n, experts))
    return (int)cudaErrorInvalidValue;
  const int chunk = plan_chunk(n), blocks = n <= chunk ? 1 : (int)(((long long)n + chunk - 1) / chunk);
  if (blocks > 1) plan_count_kernel<<<blocks, 256, experts * sizeof(int), stream>>>(indices, is_long, n, experts, chunk, workspace);
  plan_place_kernel<<<blocks, 256, (9 * (size_t)experts + 1) * sizeof(int), stream>>>(
      indices, is_long, n, experts, chunk, blocks > 1 ? workspace : nullptr, offsets, positions);
  return (int)cudaGetLastError();
}

// warps of a grid-stride kernel: up to four blocks of 8 warps per SM
static int row_blocks(long long items) { return (int)std::max<long long>(1, std::min<long long>((items + 7) / 8, 148LL * 8)); }

extern "C" int vb_expert_dispatch(const void* x, long long x_stride_bytes, long long row_bytes, int tokens, int top_k,
                                  const int* positions, const int* offsets, int experts, void* rows, cudaStream_t stream) {
  if (tokens < 0 || top_k < 1 || top_k > kMaxTopK || experts < 1 || row_bytes < 1 || row_bytes > (1LL << 24) ||
      (long long)tokens * top_k > INT_MAX)
    return (int)cudaErrorInvalidValue;
  if (tokens == 0) return 0;
  long long unit = 16;
  while (unit > 1 && (row_bytes % unit || x_stride_bytes % unit || !aligned_to(x, unit) || !aligned_to(rows, unit))) unit >>= 1;
  if (unit < 2) return (int)cudaErrorInvalidValue;
  const int words = (int)(row_bytes / unit);
  auto launch = [&](auto word) {
    using W = decltype(word);
    constexpr int U = 4;
    const int segments = (words + 32 * U - 1) / (32 * U);
    dispatch_kernel<W, U><<<row_blocks((long long)tokens * segments), 256, 0, stream>>>(
        (const W*)x, x_stride_bytes / unit, words, segments, tokens, top_k, positions, offsets, experts, (W*)rows);
  };
  if (unit == 16) launch(uint4{});
  else if (unit == 8) launch(uint2{});
  else if (unit == 4) launch(uint32_t{});
  else launch(uint16_t{});
  return (int)cudaGetLastError();
}

static bool combine_shape_ok(int dtype, int width, int tokens, int top_k, int weight_dtype) {
  return dtype >= kF32 && dtype <= kF16 && weight_dtype >= kF32 && weight_dtype <= kF16 && width >= 1 && width <= (1 << 22) &&
         tokens >= 0 && top_k >= 1 && top_k <= kMaxTopK && (long long)tokens * top_k <= INT_MAX;
}

extern "C" int vb_expert_combine(const void* rows, int dtype, int width, int tokens, int top_k, const int* positions,
                                 const void* weights, int weight_dtype, void* out, cudaStream_t stream) {
  if (!combine_shape_ok(dtype, width, tokens, top_k, weight_dtype)) return (int)cudaErrorInvalidValue;
  if (tokens == 0) return 0;
  const int size = dtype == kF32 ? 4 : 2, pack = 16 / size;
  const bool wide = width % pack == 0 && aligned_to(rows, 16) && aligned_to(out, 16);
  VB_FLOAT_SWITCH(dtype, {
    constexpr int N = 16 / (int)sizeof(T);
    if (wide) {
      const int segments = (width / N + 63) / 64;
      combine_kernel<T, N, 2><<<row_blocks((long long)tokens * segments), 256, 0, stream>>>(
          (const T*)rows, width, segments, tokens, top_k, positions, weights, weight_dtype, (T*)out);
    } else {
      const int segments = (width + 127) / 128;
      combine_kernel<T, 1, 4><<<row_blocks((long long)tokens * segments), 256, 0, stream>>>(
          (const T*)rows, width, segments, tokens, top_k, positions, weights, weight_dtype, (T*)out);
    }
  });
  return (int)cudaGetLastError();
}

extern "C" int vb_expert_combine_backward(const void* dout, const void* rows, int dtype, int width, int tokens, int top_k,
                                          const int* positions, const int* offsets, int experts, const void* weights,
                                          int weight_dtype, void* drows, void* dweights, cudaStream_t stream) {
  if (!combine_shape_ok(dtype, width, tokens, top_k, weight_dtype) || experts < 1 || (tokens > 0 && weights == nullptr))
    return (int)cudaErrorInvalidValue;
  if (tokens == 0) return 0;
  const int size = dtype == kF32 ? 4 : 2, pack = 16 / size;
  const bool wide = width % pack == 0 && aligned_to(rows, 16) && aligned_to(dout, 16) && (drows == nullptr || aligned_to(drows, 16));
  const int packs = wide ? width / pack : width;
  int team = 1;
  while (team < 8 && packs > team * 32 * 4) team *= 2;
  const int blocks = row_blocks((long long)tokens * team);
  VB_FLOAT_SWITCH(dtype, {
    constexpr int N = 16 / (int)sizeof(T);
    if (wide)
      combine_backward_kernel<T, N, 4><<<blocks, 256, 0, stream>>>((const T*)dout, (const T*)rows, width, tokens, top_k, team,
                                                                   positions, offsets, experts, weights, weight_dtype,
                                                                   (T*)drows, dweights);
    else
      combine_backward_kernel<T, 1, 4><<<blocks, 256, 0, stream>>>((const T*)dout, (const T*)rows, width, tokens, top_k, team,
                                                                   positions, offsets, experts, weights, weight_dtype,
                                                                   (T*)drows, dweights);
  });
  return (int)cudaGetLastError();
}
