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
#include "common/launch.cuh"
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

// shared memory words of a warp's lists in the forward pass, V keys a lane
__host__ __device__ constexpr int route_list_words(int v) { return ((v + 4) / 4 * 4 + (v + 3) / 4 * 4) * 32 + 64; }

template <int G, typename N> __device__ __forceinline__ N group_sum(N v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
template <int G> __device__ __forceinline__ float group_max(float v) {
  if constexpr (G == 32) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
  }
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

// Unsigned integers in the order of the keys.  A key comes out of an addition, which leaves neither -0 (the bias is never
// -0) nor a NaN with the sign set: NaN is the largest, as a descending sort has it, and nothing is below -inf.  Keys of
// -inf are never chosen, and kTaken marks those that have been.
constexpr unsigned kTaken = 0u, kClosed = 0x007fffffu;       // kClosed: ordered(-inf)
__device__ __forceinline__ unsigned ordered(float key) {
  const unsigned bits = __float_as_uint(key);
  return bits ^ ((unsigned)((int)bits >> 31) | 0x80000000u);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// e[i] = exp(l[i] - top) with top the row's maximum; returns their sum.  The hardware's base-2 exponential is off by about
// 2^-22 of its value and its argument by 2^-24 |l - top|, a few steps of fp32 where p is not negligible.  Over 131072 x 256
// fp32 logits p is off by 6.1e-8 of its norm, with expf by 5.9e-8, and the passes take 112 and 68 us, with expf 116 and 69
// (bf16: 108 and 47, 115 and 51).
template <int G, int V>
__device__ __forceinline__ float group_exp(const float (&l)[V], float (&e)[V], float& top) {
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < V; ++i) m = fmaxf(m, l[i]);
  top = group_max<G>(m);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    e[i] = exp2_fast((l[i] - top) * 1.4426950408889634f);
    s += e[i];
  }
  return group_sum<G>(s);
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

// The losses of a batch from dot = sum_e counts_e sum_t p_te, choices = sum_e counts_e (up to 32 for each of 2^31 - 1 tokens),
// z = sum of lse^2 and the tokens.
__device__ __forceinline__ void route_losses(const RouteArgs& a, float dot, long long choices, float z, int tokens) {
  const float per_token = 1.f / (float)max(tokens, 1), per_choice = 1.f / (float)max(choices, 1LL);
  *a.balance = (float)a.experts * dot * per_token * per_choice;
  *a.z = z * per_token;
  a.inverse[0] = per_token;
  a.inverse[1] = per_choice;
}

// Sorts a lane's keys, largest first: Batcher's odd-even merge sort, 19 exchanges for 8 keys, 63 for 16.
template <int V> __device__ __forceinline__ void sort_keys(unsigned (&key)[V]) {
#pragma unroll
  for (int p = 1; p < V; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < V; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const unsigned high = max(key[i + j], key[i + j + k]);
            key[i + j + k] = min(key[i + j], key[i + j + k]);
            key[i + j] = high;
          }
}

// A lane sorts its (up to 16) keys; each choice then costs one maximum over the token's lanes and one step down the winner's
// list in shared memory, and which expert a winning key belongs to is looked up for all choices at once.  More keys than
// that are searched again for every choice.
// Bound by the integer instructions it issues (131072 x 256, top 8, fp32: about 550 a token, 113 us for what 22 would
// read), many of them the same for a token whatever its experts: 16 lanes to a token put two tokens into each.  Keys
// scanned again for every choice took 226 us, sorted together with their indices 140, ranked by pairs 120.
// Four blocks an SM: 64 registers hold 16 keys a lane, and 32 warps hide the exchanges (119 us; 139 with 105 registers;
// 113 once the finishing kernel had its loads under way together).
template <typename T, int G, int V>
__global__ void __launch_bounds__(256, V <= 16 ? 4 : 2)
route_forward_kernel(const RouteArgs a) {
  cudaTriggerProgrammaticLaunchCompletion();    // the finishing kernel may start when there is room; it waits for this one
  constexpr int kWarps = 8, kThreads = kWarps * 32;
  constexpr int kTokens = 32 / G;               // tokens a warp serves at a time
  constexpr bool kSorted = V > 1 && V <= 16;
  // [experts] counts, [G * V] bias; then per warp, by lane, [V + 1][32] keys in descending order, [32][V] keys as they come,
  // [32] winning keys and [32] their lanes; in the end in their place [warps][experts] sums of p
  extern __shared__ __align__(16) unsigned char route_shared[];
  int* count = reinterpret_cast<int*>(route_shared);
  float* bias = reinterpret_cast<float*>(route_shared + (a.experts + 3) / 4 * 16);
  float* shared = bias + G * V;
  __shared__ float z_part[kWarps], dot_part[kWarps];
  __shared__ int n_part[kWarps], sum_part[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane & (G - 1), base = lane - sub;
  unsigned* lists = reinterpret_cast<unsigned*>(shared) + warp * route_list_words(V) + lane;      // [place * 32]
  uint4* keys = reinterpret_cast<uint4*>(lists - lane + (V + 4) / 4 * 4 * 32);                    // [word * 32 + lane]
  unsigned* winners = lists - lane + route_list_words(V) - 64;                                   // [32] keys, [32] lanes
  for (int e = threadIdx.x; e < G * V; e += kThreads) {
    if (e < a.experts) count[e] = 0;
    // +inf (and NaN) as the largest number, so that a logit of -inf stays closed; -0 as 0
    const float b = a.bias != nullptr && e < a.experts ? a.bias[e] : 0.f;
    bias[e] = b < INFINITY ? b + 0.f : 3.402823466e+38f;
  }
  __syncthreads();

  float p_sum[V], z_sum = 0.f;
  int live_tokens = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) p_sum[i] = 0.f;
  if constexpr (kSorted) lists[V * 32] = kTaken;                                // the end of every list
  for (long long first = (long long)(blockIdx.x * kWarps + warp) * kTokens; first < a.tokens;
       first += (long long)gridDim.x * kThreads / G) {
    const long long token = first + lane / G;
    const bool inside = token < a.tokens, live = inside && (a.mask == nullptr || a.mask[token] != 0);
    float l[V], e[V], top;
    unsigned key[V];
    if (live) {
      load_values<T, G, V>(reinterpret_cast<const T*>(a.logits) + token * a.stride, sub, a.experts, a.wide, l);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) l[i] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = ordered(l[i] + bias[sub * V + i]);
    const float total = group_exp<G, V>(l, e, top);

    int my_index = -1;
    if constexpr (kSorted) {
#pragma unroll
      for (int w = 0; w < (V + 3) / 4; ++w)
        keys[w * 32 + lane] = make_uint4(key[4 * w], 4 * w + 1 < V ? key[4 * w + 1 < V ? 4 * w + 1 : 0] : kTaken,
                                         4 * w + 2 < V ? key[4 * w + 2 < V ? 4 * w + 2 : 0] : kTaken,
                                         4 * w + 3 < V ? key[4 * w + 3 < V ? 4 * w + 3 : 0] : kTaken);
      sort_keys<V>(key);
#pragma unroll
      for (int i = 0; i < V; ++i) lists[i * 32] = key[i];
      unsigned best = key[0];
      int place = 0, found = 0;
      for (int j = 0; j < a.top_k; ++j) {
        unsigned most = best;
        if constexpr (G == 32) {
          most = __reduce_max_sync(kFull, best);
        } else {
#pragma unroll
          for (int o = G / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(kFull, most, o));
        }
        // lanes own ascending experts, so the lowest lane with the largest key has the lowest index among equals
        const unsigned holders = __ballot_sync(kFull, best == most) >> base & (G == 32 ? kFull : (1u << G) - 1u);
        const int owner = __ffs(holders) - 1;
        const bool open = most > kClosed;        // no list is at its end before a key of -inf wins
        if (sub == j) {
          winners[lane] = most;
          winners[32 + lane] = base + owner;
        }
        found += open ? 1 : 0;
        place += open && sub == owner ? 32 : 0;
        best = lists[place];
      }
      // which of its lane's keys the winner is: the first that equals it, or the next ones where the lane won with equal
      // keys.  A lane without a choice asks for a key that nothing equals, each its own.
      __syncwarp();
      const bool asks = sub < found;
      const unsigned winner = asks ? winners[lane] : kTaken;
      const int from = asks ? (int)winners[32 + lane] : lane;
      const unsigned equals = __match_any_sync(kFull, (unsigned long long)winner << 32 | (asks ? from : 32 + lane));
      int skip = __popc(equals & ((1u << lane) - 1u)), at = 0;
#pragma unroll
      for (int w = 0; w < (V + 3) / 4; ++w) {
        const uint4 word = keys[w * 32 + from];
        const unsigned v[4] = {word.x, word.y, word.z, word.w};
#pragma unroll
        for (int i = 0; i < 4 && w * 4 + i < V; ++i) {
          const bool equal = v[i] == winner;
          at = equal && skip == 0 ? w * 4 + i : at;
          skip -= equal ? 1 : 0;
        }
      }
      if (asks) my_index = (from - base) * V + at;
      __syncwarp();                              // the places are written again for the next token
    } else {
      for (int j = 0; j < a.top_k; ++j) {
        unsigned best = key[0];
#pragma unroll
        for (int i = 1; i < V; ++i) best = max(best, key[i]);
        unsigned most;
        if constexpr (G == 32) {
          most = __reduce_max_sync(kFull, best);
        } else {
          most = best;
#pragma unroll
          for (int o = G / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(kFull, most, o));
        }
        const unsigned holders = __ballot_sync(kFull, best == most) >> base & (G == 32 ? kFull : (1u << G) - 1u);
        const int owner = __ffs(holders) - 1;    // as above
        int at = 0;
#pragma unroll
        for (int i = V - 1; i >= 0; --i)
          if (key[i] == most) at = i;
        const int chosen = owner * V + __shfl_sync(kFull, at, base + owner);
        if (sub == j && most > kClosed) my_index = chosen;
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (sub * V + i == chosen) key[i] = kTaken;
      }
    }

    const bool counted = __shfl_sync(kFull, my_index, base) >= 0;
    // the row has just been read: the chosen logits come from the cache
    const float logit = my_index >= 0 ? to_float(reinterpret_cast<const T*>(a.logits)[token * a.stride + my_index]) : -INFINITY;
    float weight;
    if (a.normalize) {                          // softmax over the chosen logits = p / (sum of the chosen p)
      const float most = group_max<G>(logit);
      const float part = my_index >= 0 ? expf(logit - most) : 0.f;
      weight = part / group_sum<G>(part);
    } else {
      weight = expf(logit - top) / total;
    }
    if (inside && sub < a.top_k) {
      a.indices[token * a.top_k + sub] = my_index;
      a.weights[token * a.top_k + sub] = my_index >= 0 ? weight : 0.f;
      if (my_index >= 0) atomicAdd(&count[my_index], 1);
    }
    if (counted) {
      const float inverse = 1.f / total, lse = top + logf(total);
#pragma unroll
      for (int i = 0; i < V; ++i) p_sum[i] = fmaf(e[i], inverse, p_sum[i]);
      if (sub == 0) {
        z_sum = fmaf(lse, lse, z_sum);
        ++live_tokens;
      }
    }
  }

  __syncthreads();                              // the lists are done with
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
  float* mine = a.partial + (long long)blockIdx.x * (2 * a.experts + 2);
  float dot = 0.f;
  int choices = 0;
  for (int e = threadIdx.x; e < a.experts; e += kThreads) {
    float total = 0.f;
    for (int w = 0; w < kWarps; ++w) total += shared[w * a.experts + e];
    if (gridDim.x > 1) {
      mine[e] = total;
      mine[a.experts + e] = __int_as_float(count[e]);
    } else {
      a.counts[e] = count[e];
      dot = fmaf((float)count[e], total, dot);
      choices += count[e];
    }
  }
  if (gridDim.x == 1) {
    dot = group_sum<32>(dot);
    choices = __reduce_add_sync(kFull, choices);
    if (lane == 0) {
      dot_part[warp] = dot;
      sum_part[warp] = choices;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    float z = 0.f;
    int n = 0;
    dot = 0.f;
    choices = 0;
    for (int w = 0; w < kWarps; ++w) {
      z += z_part[w];
      n += n_part[w];
      if (gridDim.x == 1) {
        dot += dot_part[w];
        choices += sum_part[w];
      }
    }
    if (gridDim.x == 1) {
      route_losses(a, dot, choices, z, n);
    } else {
      mine[2 * a.experts] = z;
      mine[2 * a.experts + 1] = __int_as_float(n);
    }
  }
}

// Adds the blocks' sums in block order and derives the losses: one cluster, each block of which takes every eighth set of
// 32 experts with 32 threads per expert; the first block adds the clusters' shares of the balance in order.
constexpr int kFinishBlocks = 8;
constexpr int kAhead = 8;                       // loads under way; they bound it
__global__ void __cluster_dims__(kFinishBlocks, 1, 1) __launch_bounds__(1024)
route_finish_kernel(const RouteArgs a, int blocks) {
  __shared__ float p_part[32][33];
  __shared__ int c_part[32][33];
  __shared__ float dot_share;                   // this block's parts of dot and of choices
  __shared__ long long choices_share;
  __shared__ float z_part[32];
  __shared__ int n_part[32];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int pitch = 2 * a.experts + 2;          // (592 sets at most)
  cudaGridDependencySynchronize();
  float dot = 0.f, z = 0.f;
  long long choices = 0;
  int n = 0;
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b < blocks; b += 1024) {
      z += a.partial[b * pitch + 2 * a.experts];
      n += __float_as_int(a.partial[b * pitch + 2 * a.experts + 1]);
    }
    z = group_sum<32>(z);
    n = __reduce_add_sync(kFull, n);
    if (lane == 0) {
      z_part[row] = z;
      n_part[row] = n;
    }
    __syncthreads();
  }
  for (int first = blockIdx.x * 32; first < a.experts; first += kFinishBlocks * 32) {
    const int e = first + lane;
    float p = 0.f;
    int c = 0;
    // places past the end read the last set's or the last expert's, so that no load waits for a condition (146 us in place of
    // 157 for 32768 x 1024 fp32, forward)
    const int column = min(e, a.experts - 1);
    for (int b = row; b < blocks; b += 32 * kAhead) {
      float ps[kAhead];
      int cs[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const float* at = a.partial + (min(b + 32 * k, blocks - 1) * pitch + column);
        ps[k] = at[0];
        cs[k] = __float_as_int(at[a.experts]);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        p += b + 32 * k < blocks ? ps[k] : 0.f;
        c += b + 32 * k < blocks ? cs[k] : 0;
      }
    }
    if (e >= a.experts) {
      p = 0.f;
      c = 0;
    }
    p_part[row][lane] = p;
    c_part[row][lane] = c;
    __syncthreads();
    if (row == 0) {
      p = 0.f;
      c = 0;
#pragma unroll 8
      for (int r = 0; r < 32; ++r) {
        p += p_part[r][lane];
        c += c_part[r][lane];
      }
      if (e < a.experts) a.counts[e] = c;
      dot += group_sum<32>((float)c * p);
      choices += c;                             // of the lane's experts
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && row == 0) {
    z = group_sum<32>(z_part[lane]);
    n = __reduce_add_sync(kFull, n_part[lane]);
  }
  if (row == 0) choices = group_sum<32>(choices);
  if (threadIdx.x == 0) {
    dot_share = dot;
    choices_share = choices;
  }
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    dot = 0.f;
    choices = 0;
    for (int b = 0; b < kFinishBlocks; ++b) {
      uint32_t at_dot, at_choices;
      float part;
      long long sum;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at_dot) : "r"((uint32_t)__cvta_generic_to_shared(&dot_share)), "r"(b));
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at_choices) : "r"((uint32_t)__cvta_generic_to_shared(&choices_share)), "r"(b));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part) : "r"(at_dot) : "memory");
      asm volatile("ld.shared::cluster.s64 %0, [%1];" : "=l"(sum) : "r"(at_choices) : "memory");
      dot += part;
      choices += sum;
    }
    route_losses(a, dot, choices, z, n);
  }
  // the others' shared memory stays until it has been read
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
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
// The softmax is formed again from the logits: reading them costs what reading a saved p would.  131072 x 256 fp32: 68 us,
// 63 % of the copy rate; before the last steps 80 at two blocks an SM and 70 at four, and 77 with the chosen experts' own terms
// by shuffles in place of shared memory.  A lane's V consecutive values put its 16-byte words V values from its neighbours'
// and its reads of `mine` into few banks (the same in bf16: 47 %, 32768 x 1024 fp32: 30 %).
template <typename T, int G, int V>
__global__ void __launch_bounds__(256, V <= 16 ? 4 : 2)
route_backward_kernel(const RouteBackwardArgs a) {
  constexpr int kTokens = 32 / G;
  __shared__ float chosen_grad[8][32 * V];      // of the tokens that a warp works on, zero where not chosen
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane & (G - 1), base = lane - sub;
  float* mine = chosen_grad[warp] + base * V;
  for (int i = lane; i < 32 * V; i += 32) chosen_grad[warp][i] = 0.f;
  __syncwarp();
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
    float l[V], p[V], top;
    if (counted) {
      load_values<T, G, V>(reinterpret_cast<const T*>(a.logits) + token * a.stride, sub, a.experts, a.wide, l);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) l[i] = -INFINITY;
    }
    const float total = group_exp<G, V>(l, p, top), lse = top + logf(total), inverse = 1.f / total;
    float pf = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      p[i] *= inverse;
      pf = fmaf(p[i], f[i], pf);
    }
    pf = group_sum<G>(pf);
    const float dot = group_sum<G>(w * g);
    const float common = cz * lse - (a.normalize ? 0.f : dot);
    const float own = w * (a.normalize ? g - dot : g);
    float grad[V];
#pragma unroll
    for (int i = 0; i < V; ++i) grad[i] = p[i] * fmaf(cb, f[i] - pf, common);
    if (index >= 0) mine[index] = own;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < V; ++i) grad[i] += mine[sub * V + i];
    __syncwarp();
    if (index >= 0) mine[index] = 0.f;
    __syncwarp();
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
// Every block owns `chunk` consecutive choices, every warp of it an equal consecutive part.  A block's first row for an
// expert is what earlier experts hold altogether plus what earlier blocks hold of this one: every block adds up all
// histograms (they stay in the second-level cache), which costs less than a third launch that would do it once.
// 32768 x 4 choices of 128 experts take 10 us, two launches one after the other; 131072 x 8 of 256 take 21, as every block adds
// 148 histograms of 256 and a warp ranks its choices 32 at a time (a thread per four experts: 14 and 45).
__device__ __forceinline__ int read_choice(const void* indices, int is_long, long long i, int experts) {
  const long long e = is_long ? reinterpret_cast<const long long*>(indices)[i] : (long long)reinterpret_cast<const int*>(indices)[i];
  return e >= 0 && e < experts ? (int)e : -1;
}

__global__ void __launch_bounds__(512)
plan_count_kernel(const void* __restrict__ indices, int is_long, int n, int experts, int chunk, int* __restrict__ histogram) {
  extern __shared__ int plan_shared[];
  for (int e = threadIdx.x; e < experts; e += 512) plan_shared[e] = 0;
  __syncthreads();
  const long long first = (long long)blockIdx.x * chunk, last = min(first + chunk, (long long)n);
#pragma unroll 8
  for (long long i = first + threadIdx.x; i < last; i += 512) {
    const int e = read_choice(indices, is_long, i, experts);
    if (e >= 0) atomicAdd(&plan_shared[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += 512) histogram[(long long)blockIdx.x * experts + e] = plan_shared[e];
}

// `columns`: experts rounded up to a power of two, at least 32; the threads form rows of that many (512 threads and more
// columns: a thread takes several)
template <int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
plan_place_kernel(const void* __restrict__ indices, int is_long, int n, int experts, int columns, int chunk,
                  const int* __restrict__ histogram, int* __restrict__ offsets, int* __restrict__ positions) {
  constexpr int kThreads = WARPS * 32;
  extern __shared__ int plan_shared[];          // [WARPS][experts] next row of every warp, [experts] totals, [experts] before
  __shared__ int scan_part[WARPS], base_part;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int* total = plan_shared + WARPS * experts;
  int* before = total + experts;
  int* next = plan_shared + warp * experts;
  for (int i = threadIdx.x; i < (WARPS + 2) * experts; i += kThreads) plan_shared[i] = 0;
  __syncthreads();
  const long long block_first = (long long)blockIdx.x * chunk, block_last = min(block_first + chunk, (long long)n);
  const long long first = block_first + (long long)warp * (chunk / WARPS), last = min(first + chunk / WARPS, block_last);
#pragma unroll 4
  for (long long i = first + lane; i < last; i += 32) {
    const int e = read_choice(indices, is_long, i, experts);
    if (e >= 0) atomicAdd(&next[e], 1);
  }
  if (histogram != nullptr) {
    const int rows = max(kThreads / columns, 1), row = threadIdx.x / columns;
    for (int e = threadIdx.x % columns; e < experts; e += kThreads) {
      int sum = 0, early = 0;
#pragma unroll 8
      for (int b = row; b < (int)gridDim.x; b += rows) {
        const int c = histogram[(long long)b * experts + e];
        sum += c;
        early += b < (int)blockIdx.x ? c : 0;
      }
      if (sum) atomicAdd(&total[e], sum);        // whole numbers: any order gives the same
      if (early) atomicAdd(&before[e], early);
    }
  }
  __syncthreads();
  if (histogram == nullptr) {
    for (int e = threadIdx.x; e < experts; e += kThreads) {
      int sum = 0;
      for (int w = 0; w < WARPS; ++w) sum += plan_shared[w * experts + e];
      total[e] = sum;
    }
  }
  // exclusive scan of the totals, a thread for every expert, kThreads experts at a time
  int carry = 0;
  for (int e0 = 0; e0 < experts; e0 += kThreads) {
    const int e = e0 + threadIdx.x, mine = e < experts ? total[e] : 0;
    int scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(kFull, scan, o);
      if (lane >= o) scan += other;
    }
    if (lane == 31) scan_part[warp] = scan;
    __syncthreads();
    int start = carry + scan - mine;
    for (int w = 0; w < warp; ++w) start += scan_part[w];
    if (e < experts) {
      int row = start + before[e];
      for (int w = 0; w < WARPS; ++w) {           // turn the warps' counts into their first rows
        const int c = plan_shared[w * experts + e];
        plan_shared[w * experts + e] = row;
        row += c;
      }
      if (blockIdx.x == 0) {
        offsets[e] = start;
        if (e == experts - 1) offsets[experts] = start + mine;
      }
    }
    if (threadIdx.x == kThreads - 1) base_part = start + mine;
    __syncthreads();
    carry = base_part;
  }
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

// One warp per (token, segment of 32 * U words): the token's words are read once and stored top_k times.  Bound by memory:
// 32768 x 2048 bf16 to four experts 105 us, 97 % of the copy rate.
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

// out[t] = sum_j weights[t, j] * rows[positions[t, j]], added in fp32 in the order of j; weights null: all one.
// A warp per (token, segment of 32 * U packs).  Bound by memory: 32768 x 2048 bf16, four choices, 106 us (96 % of the copy
// rate); threads over the flattened result instead of warps over rows took 158.
template <typename T, int N, int U>
__global__ void __launch_bounds__(256, 2)
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
// A token is served by `team` warps of a block (1, 2, 4 or 8) with up to U packs a lane in flight; after the first choice
// its row of dout comes from the cache, and the dot products end in the block.
// 32768 tokens x 1152 bf16, two choices: 94 us with two warps of four packs that split a row unevenly, 77 us evenly, 64 us
// with one warp of five (90 % of the copy rate).  Bound by loads in flight: at 2 blocks an SM instead of 3 or 4 it took 109.
template <typename T, int N, int U>
__global__ void __launch_bounds__(256, U <= 4 ? 4 : 3)
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
          // the warps of a team take every team-th stretch of 32 packs
          for (int first = (member * 32 + lane) * N; first < width; first += team * 32 * U * N) {
            Pack<T, N> g[U], v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int c = first + 32 * u * team * N;
              if (c < width) {
                v[u].load(rows + (long long)row * width + c);
                g[u].load(dout + token * width + c);
              }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int c = first + 32 * u * team * N;
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

extern "C" long long vb_block_launches(void) { return launches.load(std::memory_order_relaxed); }

static bool aligned_to(const void* p, long long bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// lanes per token (G) and experts per lane (V)
#define VB_ROUTE_CASE(g, v, ...) if (lanes == g && per_lane == v) { constexpr int G = g, V = v; __VA_ARGS__; }
#define VB_ROUTE_SWITCH(...)                                                                     \
  VB_ROUTE_CASE(4, 1, __VA_ARGS__) else VB_ROUTE_CASE(8, 1, __VA_ARGS__)                         \
  else VB_ROUTE_CASE(16, 1, __VA_ARGS__) else VB_ROUTE_CASE(16, 2, __VA_ARGS__)                  \
  else VB_ROUTE_CASE(16, 4, __VA_ARGS__) else VB_ROUTE_CASE(16, 8, __VA_ARGS__)                  \
  else VB_ROUTE_CASE(16, 16, __VA_ARGS__) else VB_ROUTE_CASE(32, 1, __VA_ARGS__)                 \
  else VB_ROUTE_CASE(32, 2, __VA_ARGS__) else VB_ROUTE_CASE(32, 4, __VA_ARGS__)                  \
  else VB_ROUTE_CASE(32, 8, __VA_ARGS__) else VB_ROUTE_CASE(32, 16, __VA_ARGS__)                 \
  else VB_ROUTE_CASE(32, 32, __VA_ARGS__)

#define VB_FLOAT_SWITCH(dtype, ...)                                              \
  if ((dtype) == kF32) { using T = float; __VA_ARGS__; }                         \
  else if ((dtype) == kBF16) { using T = __nv_bfloat16; __VA_ARGS__; }           \
  else { using T = __half; __VA_ARGS__; }

// A token's lanes hold one choice each at the end, so there are at least top_k of them.
static int route_lanes(int experts, int top_k) {
  if (experts <= 16) return experts <= 4 ? 4 : experts <= 8 ? 8 : 16;
  return top_k <= 16 && experts <= 256 ? 16 : 32;
}
static int route_per_lane(int experts, int lanes) {
  int v = 1;
  while (v * lanes < experts) v *= 2;
  return v;
}
// Blocks (of 8 warps) of the forward pass: one where it makes no more than four passes, else at most four per SM
static int route_blocks(int tokens, int lanes) {
  const long long per_pass = 8LL * (32 / lanes);
  if (tokens <= 4 * per_pass) return 1;
  return (int)std::min<long long>((tokens + per_pass - 1) / per_pass, 148LL * 4);
}
static bool route_wide(const void* p, long long stride, int experts, int lanes, int per_lane, int size) {
  const int bytes = std::min(16, per_lane * size);
  return experts == lanes * per_lane && aligned_to(p, bytes) && stride * size % bytes == 0;
}
static bool route_shape_ok(int tokens, int experts, int top_k, int dtype) {
  return tokens >= 0 && experts >= 1 && experts <= kMaxExperts && top_k >= 1 && top_k <= std::min(experts, kMaxTopK) &&
         dtype >= kF32 && dtype <= kF16;
}

// (for any top_k: 16 lanes make the fewest tokens per pass for short batches, 32 the most blocks)
extern "C" long long vb_route_workspace(int tokens, int experts) {
  if (tokens < 0 || experts < 1) return 0;
  return (long long)std::max(route_blocks(tokens, route_lanes(experts, 1)), route_blocks(tokens, route_lanes(experts, kMaxTopK))) *
         (2 * experts + 2);
}

extern "C" int vb_route_forward(const void* logits, int dtype, int tokens, int experts, long long stride, const float* bias,
                                const uint8_t* mask, int top_k, int normalize, float* weights, int* indices, int* counts,
                                float* balance, float* z, float* inverse, float* workspace, long long workspace_floats,
                                cudaStream_t stream) {
  if (!route_shape_ok(tokens, experts, top_k, dtype) || workspace == nullptr ||
      workspace_floats < vb_route_workspace(tokens, experts))
    return (int)cudaErrorInvalidValue;
  const int lanes = route_lanes(experts, top_k), per_lane = route_per_lane(experts, lanes), blocks = route_blocks(tokens, lanes);
  RouteArgs a{logits, stride, tokens, experts, top_k, normalize, 0, bias, mask, weights, indices, counts, balance, z, inverse,
              workspace};
  a.wide = route_wide(logits, stride, experts, lanes, per_lane, dtype == kF32 ? 4 : 2);
  const size_t lists = per_lane > 1 && per_lane <= 16 ? 8 * route_list_words(per_lane) * sizeof(int) : 0;
  // at most 42 KB: 512 experts in 32 lanes of 16 keys
  static_assert(8 * route_list_words(16) * 4 + 2 * 512 * 4 <= 47 * 1024 && 8 * kMaxExperts * 4 + 2 * kMaxExperts * 4 <= 47 * 1024,
                "beyond what a kernel has without asking for more");
  const size_t smem = ((size_t)(experts + 3) / 4 * 4 + lanes * per_lane) * 4 + std::max(lists, (size_t)8 * experts * sizeof(float));
  VB_FLOAT_SWITCH(dtype, VB_ROUTE_SWITCH((route_forward_kernel<T, G, V><<<blocks, 256, smem, stream>>>(a))));
  count_launch();
  if (blocks > 1) launch_early(route_finish_kernel, kFinishBlocks, 1024, 0, stream, a, blocks);
  return (int)cudaGetLastError();
}

extern "C" int vb_route_backward(const void* logits, int dtype, int tokens, int experts, long long stride, int top_k,
                                 int normalize, const float* weights, const int* indices, const int* counts,
                                 const float* inverse, const float* dweights, const float* dbalance, const float* dz,
                                 void* dlogits, cudaStream_t stream) {
  if (!route_shape_ok(tokens, experts, top_k, dtype)) return (int)cudaErrorInvalidValue;
  if (tokens == 0) return 0;
  const int lanes = route_lanes(experts, top_k), per_lane = route_per_lane(experts, lanes), size = dtype == kF32 ? 4 : 2;
  RouteBackwardArgs a{logits, stride, tokens, experts, top_k, normalize, 0, weights, indices, counts, inverse, dweights,
                      dbalance, dz, dlogits};
  a.wide = route_wide(logits, stride, experts, lanes, per_lane, size) && route_wide(dlogits, experts, experts, lanes, per_lane, size);
  const long long per_pass = 8LL * (32 / lanes);
  const int blocks = (int)std::min<long long>((tokens + per_pass - 1) / per_pass, 148LL * 8);
  VB_FLOAT_SWITCH(dtype, VB_ROUTE_SWITCH((route_backward_kernel<T, G, V><<<blocks, 256, 0, stream>>>(a))));
  count_launch();
  return (int)cudaGetLastError();
}

// choices per block: a multiple of 16 warps x 32 lanes; about one block per SM for long lists
static int plan_chunk(int n) {
  const long long per = ((long long)n + 147) / 148;
  return (int)std::max<long long>(4096, (per + 511) / 512 * 512);
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
  int columns = 32;
  while (columns < experts) columns *= 2;
  if (blocks > 1) {
    plan_count_kernel<<<blocks, 512, experts * sizeof(int), stream>>>(indices, is_long, n, experts, chunk, workspace);
    count_launch();
  }
  const int* histogram = blocks > 1 ? workspace : nullptr;
  if (experts <= 512)
    plan_place_kernel<16><<<blocks, 512, 18 * (size_t)experts * sizeof(int), stream>>>(indices, is_long, n, experts, columns, chunk,
                                                                                      histogram, offsets, positions);
  else                                           // 8 warps' counts of more experts fit 48 KB
    plan_place_kernel<8><<<blocks, 256, 10 * (size_t)experts * sizeof(int), stream>>>(indices, is_long, n, experts, columns, chunk,
                                                                                     histogram, offsets, positions);
  count_launch();
  return (int)cudaGetLastError();
}

// Blocks of 8 warps for so many items of a warp.  32 blocks an SM, four times what is resident, even out the tail of long
// runs: dispatch of 32768 x 2048 bf16 to four experts 113 us at 8 blocks an SM, 107 us at 32 in the same run.
static int row_blocks(long long items) {
  const long long most = items >= 148LL * 32 * 8 ? 148 * 32 : 148 * 8;
  return (int)std::max<long long>(1, std::min<long long>((items + 7) / 8, most));
}
// Packs a lane: a whole row (up to 8 a lane) to a warp where that leaves every SM 16 warps, so that all its loads are in
// flight together, else 2.  32768 x 1152 bf16, two choices: combine 52 us at 2 a lane, 45 us at 5; 32768 x 2048, four choices:
// 120 at 2, 106 at 8.
static int row_packs(int packs, int tokens) {
  if (tokens < 148 * 16) return 2;
  const int segments = (packs + 255) / 256, per_lane = (packs + segments * 32 - 1) / (segments * 32);
  return per_lane <= 2 ? 2 : per_lane <= 5 ? 5 : 8;
}

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
  count_launch();
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
  const int packs = wide ? width / pack : width, per_lane = row_packs(packs, tokens);
  const int segments = (packs + per_lane * 32 - 1) / (per_lane * 32), blocks = row_blocks((long long)tokens * segments);
  VB_FLOAT_SWITCH(dtype, {
    constexpr int N = 16 / (int)sizeof(T);
    auto launch = [&](auto kernel) {
      kernel<<<blocks, 256, 0, stream>>>((const T*)rows, width, segments, tokens, top_k, positions, weights, weight_dtype, (T*)out);
    };
    if (wide && per_lane == 2) launch(combine_kernel<T, N, 2>);
    else if (wide && per_lane == 5) launch(combine_kernel<T, N, 5>);
    else if (wide) launch(combine_kernel<T, N, 8>);
    else if (per_lane == 2) launch(combine_kernel<T, 1, 2>);
    else if (per_lane == 5) launch(combine_kernel<T, 1, 5>);
    else launch(combine_kernel<T, 1, 8>);
  });
  count_launch();
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
  // (at most 5 packs a lane: 32768 x 2048 bf16, four choices, 199 us with two warps of four, 249 with one of eight)
  const int packs = wide ? width / pack : width, most = std::min(5, row_packs(packs, tokens));
  int team = 1;
  while (team < 8 && packs > team * 32 * most) team *= 2;
  const int per_lane = (packs + team * 32 - 1) / (team * 32), blocks = row_blocks((long long)tokens * team);
  VB_FLOAT_SWITCH(dtype, {
    constexpr int N = 16 / (int)sizeof(T);
    auto launch = [&](auto kernel) {
      kernel<<<blocks, 256, 0, stream>>>((const T*)dout, (const T*)rows, width, tokens, top_k, team, positions, offsets, experts,
                                         weights, weight_dtype, (T*)drows, dweights);
    };
    if (wide && per_lane <= 2) launch(combine_backward_kernel<T, N, 2>);
    else if (wide && per_lane <= 4) launch(combine_backward_kernel<T, N, 4>);
    else if (wide) launch(combine_backward_kernel<T, N, 5>);
    else if (per_lane <= 2) launch(combine_backward_kernel<T, 1, 2>);
    else launch(combine_backward_kernel<T, 1, 4>);
  });
  count_launch();
  return (int)cudaGetLastError();
}
