// RMS norms after and before a transformer block, fused with the block's gate and the residual scale:
//
//   yh  = y * ry,  ry = (mean(y^2) + eps)^-1/2              (POST: the norm after the block)
//   u   = alpha * x + gate * weight * yh                    -> out, the residual stream
//   h   = u * ru * next_weight * (1 + next_scale)           (PRE: the norm before the next block; u = x without POST)
//
// One pass each way: a row's values stay in registers between the statistics and the results, and the backward pass
// forms u again from x and y, which the graph holds anyway, so nothing but the two reciprocal roots is saved.
// Vectors are fp32, bf16 or fp16 with a pitch per sample (0: one vector for all rows); all arithmetic is fp32.
#include <climits>

#include "api.h"
#include "common/numerics.cuh"

namespace vb {

constexpr unsigned kAll = 0xffffffffu;

struct NormVector {            // [samples, cols] (or [cols] with pitch 0), null = absent
  const void* data;
  int dtype;
  long long pitch;
};
struct NormArgs {
  int rows, cols, tokens;      // tokens: rows of a sample
  int warps;                   // warps of a row
  float alpha, eps;
  const void *x, *y;
  NormVector weight, gate, next_weight, next_scale;
  void *out, *h;
  float *ry, *ru;              // forward: written when not null; backward: read
  // backward
  const void *dout, *dh;       // either may be null
  void *dx, *dy;               // either may be null
  int units_per_sample;        // row sets that a sample's column sums are split into
  float* sums;                 // [samples * units_per_sample][2][cols]: sums of d * yh and of dh * uh, or null
};

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void assign(float& to, float v) { to = v; }
__device__ __forceinline__ void assign(__nv_bfloat16& to, float v) { to = __float2bfloat16_rn(v); }
__device__ __forceinline__ void assign(__half& to, float v) { to = __float2half_rn(v); }

// VEC neighbouring values as they are stored
template <typename T, int VEC> struct Piece {
  static constexpr int kBytes = VEC * (int)sizeof(T);
  static constexpr bool kWide = kBytes >= 16;
  union {
    T value[VEC];
    uint4 word[kWide ? kBytes / 16 : 1];
  };
  __device__ __forceinline__ Piece() {}
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kWide) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) word[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) value[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kWide) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(p)[i] = word[i];
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) p[i] = value[i];
    }
  }
  __device__ __forceinline__ float get(int i) const { return as_float(value[i]); }
  __device__ __forceinline__ void set(int i, float v) { assign(value[i], v); }
};

// Sums N values over the warps of a row; every thread gets them.  `turn` alternates between two buffers, so that one
// barrier per call is enough: a warp can only reach the buffer's next use through the other buffer's barrier.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int warps, float (*buffer)[32][N], int& turn) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[n] += __shfl_xor_sync(kAll, v[n], o);
  if (warps == 1) return;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) buffer[turn][threadIdx.x >> 5][n] = v[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = 0.f;
  for (int w = 0; w < warps; ++w)
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += buffer[turn][w][n];
  turn ^= 1;
}

// product of two optional vectors (the second as 1 + v when `shifted`) for the columns of one thread
template <int VEC, int V>
__device__ __forceinline__ void load_gain(const NormVector& a, const NormVector& b, bool shifted, int sample, int tid,
                                          int threads, int cols, float (&gain)[V][VEC]) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (tid + j * threads) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float g = 1.f;
      if (c < cols) {
        if (a.data != nullptr) g = load_as_float(a.data, sample * a.pitch + c + i, a.dtype);
        if (b.data != nullptr) g *= (shifted ? 1.f : 0.f) + load_as_float(b.data, sample * b.pitch + c + i, b.dtype);
      }
      gain[j][i] = g;
    }
  }
}

template <typename TX, typename TY, int VEC, int V, bool POST, bool PRE>
__global__ void __launch_bounds__(VEC == 1 ? 1024 : 512)
norm_forward_kernel(const NormArgs a) {
  __shared__ float buffer[2][32][1];
  const int threads = a.warps * 32, group = threadIdx.x / threads, tid = threadIdx.x - group * threads;
  const int groups = blockDim.x / threads, units = gridDim.x * groups;
  const int per_unit = (a.rows + units - 1) / units;
  const long long first = (long long)(blockIdx.x * groups + group) * per_unit;
  const int last = (int)min(first + per_unit, (long long)a.rows);
  const TX* x = reinterpret_cast<const TX*>(a.x);
  const TY* y = reinterpret_cast<const TY*>(a.y);
  const float inverse = 1.f / (float)a.cols;
  float gain[V][VEC], next_gain[V][VEC];
  int sample = -1, turn = 0;
  for (long long row = first; row < last; ++row) {
    if ((int)(row / a.tokens) != sample) {
      sample = (int)(row / a.tokens);
      if (POST) load_gain<VEC, V>(a.weight, a.gate, false, sample, tid, threads, a.cols, gain);
      if (PRE) load_gain<VEC, V>(a.next_weight, a.next_scale, true, sample, tid, threads, a.cols, next_gain);
    }
    const long long base = row * a.cols;
    Piece<TX, VEC> px[V];
    Piece<TY, VEC> py[V];
    float u[V][VEC], sum[1] = {0.f};
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (tid + j * threads) * VEC;
      if (c < a.cols) {
        px[j].load(x + base + c);
        if (POST) py[j].load(y + base + c);
      }
    }
    if (POST) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if ((tid + j * threads) * VEC < a.cols)
#pragma unroll
          for (int i = 0; i < VEC; ++i) sum[0] = fmaf(py[j].get(i), py[j].get(i), sum[0]);
      row_sum<1>(sum, a.warps, buffer, turn);
      const float ry = rsqrtf(fmaf(sum[0], inverse, a.eps));
      if (tid == 0 && a.ry != nullptr) a.ry[row] = ry;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = (tid + j * threads) * VEC;
        if (c < a.cols) {
          Piece<TX, VEC> o;
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            u[j][i] = fmaf(a.alpha, px[j].get(i), py[j].get(i) * ry * gain[j][i]);
            o.set(i, u[j][i]);
          }
          o.store(reinterpret_cast<TX*>(a.out) + base + c);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) u[j][i] = px[j].get(i);
    }
    if (PRE) {
      sum[0] = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if ((tid + j * threads) * VEC < a.cols)
#pragma unroll
          for (int i = 0; i < VEC; ++i) sum[0] = fmaf(u[j][i], u[j][i], sum[0]);
      row_sum<1>(sum, a.warps, buffer, turn);
      const float ru = rsqrtf(fmaf(sum[0], inverse, a.eps));
      if (tid == 0 && a.ru != nullptr) a.ru[row] = ru;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = (tid + j * threads) * VEC;
        if (c < a.cols) {
          Piece<TY, VEC> o;
#pragma unroll
          for (int i = 0; i < VEC; ++i) o.set(i, u[j][i] * ru * next_gain[j][i]);
          o.store(reinterpret_cast<TY*>(a.h) + base + c);
        }
      }
    }
  }
}

// With q = gate * weight * yh, t = dh * next_weight * (1 + next_scale), uh = u * ru, c = mean(t uh):
//   d  = dout + ru (t - uh c)                  the gradient of u
//   dx = alpha d,   dy = ry (d gate weight - yh m),   m = mean(d q)
// mean(d q) = mean((dout + ru t) q) - ru c mean(uh q), so one reduction of three sums per row serves both norms.
// A unit (a block, or a warp where a row takes one) walks every units_per_sample-th row of one sample and keeps the
// column sums of d * yh and dh * uh; they are parked in `sums` and added in unit order by norm_sums_kernel.
template <typename TX, typename TY, int VEC, int V, bool POST, bool PRE>
__global__ void __launch_bounds__(VEC == 1 ? 1024 : 512)
norm_backward_kernel(const NormArgs a) {
  __shared__ float buffer[2][32][3];
  const int threads = a.warps * 32, group = threadIdx.x / threads, tid = threadIdx.x - group * threads;
  const int groups = blockDim.x / threads;
  const long long unit = (long long)blockIdx.x * groups + group;
  const long long sample = unit / a.units_per_sample;
  if (sample * a.tokens >= a.rows) return;      // only where a row takes one warp: no barrier follows
  const long long end = min((sample + 1) * a.tokens, (long long)a.rows);
  const TX* x = reinterpret_cast<const TX*>(a.x);
  const TY* y = reinterpret_cast<const TY*>(a.y);
  const TX* dout = reinterpret_cast<const TX*>(a.dout);
  const TY* dh = reinterpret_cast<const TY*>(a.dh);
  const float inverse = 1.f / (float)a.cols;
  float gain[V][VEC], next_gain[V][VEC], post_sum[V][VEC], pre_sum[V][VEC];
  if (POST) load_gain<VEC, V>(a.weight, a.gate, false, (int)sample, tid, threads, a.cols, gain);
  if (PRE) load_gain<VEC, V>(a.next_weight, a.next_scale, true, (int)sample, tid, threads, a.cols, next_gain);
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int i = 0; i < VEC; ++i) post_sum[j][i] = pre_sum[j][i] = 0.f;
  int turn = 0;
  for (long long row = sample * a.tokens + unit % a.units_per_sample; row < end; row += a.units_per_sample) {
    const long long base = row * a.cols;
    const float ry = POST ? a.ry[row] : 0.f, ru = PRE ? a.ru[row] : 0.f;
    float d[V][VEC], yh[V][VEC], uh[V][VEC], sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (tid + j * threads) * VEC;
      Piece<TX, VEC> px, pd;
      Piece<TY, VEC> py, ph;
      if (c < a.cols) {
        if (PRE) px.load(x + base + c);
        if (POST) py.load(y + base + c);
        if (a.dout != nullptr) pd.load(dout + base + c);
        if (PRE) ph.load(dh + base + c);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float q = 0.f, u;
          d[j][i] = a.dout != nullptr ? pd.get(i) : 0.f;
          if (POST) {
            yh[j][i] = py.get(i) * ry;
            q = yh[j][i] * gain[j][i];
          }
          if (PRE) {
            u = POST ? fmaf(a.alpha, px.get(i), q) : px.get(i);
            uh[j][i] = u * ru;
            const float g = ph.get(i), t = g * next_gain[j][i];
            pre_sum[j][i] = fmaf(g, uh[j][i], pre_sum[j][i]);
            sum[0] = fmaf(t, uh[j][i], sum[0]);
            d[j][i] = fmaf(ru, t, d[j][i]);
            if (POST) sum[2] = fmaf(uh[j][i], q, sum[2]);
          }
          if (POST) sum[1] = fmaf(d[j][i], q, sum[1]);
        }
      }
    }
    row_sum<3>(sum, a.warps, buffer, turn);
    const float pull = ru * sum[0] * inverse;                       // ru c
    const float m = POST ? (PRE ? fmaf(-pull, sum[2], sum[1]) : sum[1]) * inverse : 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (tid + j * threads) * VEC;
      if (c < a.cols) {
        Piece<TX, VEC> ox;
        Piece<TY, VEC> oy;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float total = PRE ? fmaf(-pull, uh[j][i], d[j][i]) : d[j][i];
          ox.set(i, POST ? a.alpha * total : total);
          if (POST) {
            oy.set(i, ry * fmaf(-m, yh[j][i], total * gain[j][i]));
            post_sum[j][i] = fmaf(total, yh[j][i], post_sum[j][i]);
          }
        }
        if (a.dx != nullptr) ox.store(reinterpret_cast<TX*>(a.dx) + base + c);
        if (POST && a.dy != nullptr) oy.store(reinterpret_cast<TY*>(a.dy) + base + c);
      }
    }
  }
  if (a.sums != nullptr) {
    float* mine = a.sums + unit * 2 * a.cols;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (tid + j * threads) * VEC;
      if (c < a.cols) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          mine[c + i] = POST ? post_sum[j][i] : 0.f;
          mine[a.cols + c + i] = PRE ? pre_sum[j][i] : 0.f;
        }
      }
    }
  }
}

struct NormSumArgs {
  int cols, samples, units_per_sample;
  const float* sums;
  NormVector factor[2][2];     // [norm][0: weight, 1: gate / next_scale]
  void* grad[2][2];            // gradients of the same, or null
};

// Gradients of the vectors from the units' column sums s: with `other` the vector's partner (1 + next_scale for
// next_weight), a per-sample vector gets other_b * sum over the sample's units, a shared one sum over all units of
// other_b * s.  Block (slot, 32 columns): slot < samples writes the per-sample vectors of that sample, the last slot the
// shared ones.  Eight threads per column take every eighth unit; their sums are added in order.
__global__ void __launch_bounds__(256)
norm_sums_kernel(const NormSumArgs a) {
  __shared__ float part[4][8][32];
  const int lane = threadIdx.x & 31, part_index = threadIdx.x >> 5, c = blockIdx.y * 32 + lane;
  const bool shared_slot = (int)blockIdx.x == a.samples;
  const long long first = shared_slot ? 0 : (long long)blockIdx.x * a.units_per_sample;
  const long long last = shared_slot ? (long long)a.samples * a.units_per_sample : first + a.units_per_sample;
  float total[2][2] = {};
  if (c < a.cols) {
    for (long long u = first + part_index; u < last; u += 8) {
      const long long sample = u / a.units_per_sample;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const NormVector &w = a.factor[n][0], &s = a.factor[n][1];
        if (a.grad[n][0] == nullptr && a.grad[n][1] == nullptr) continue;
        const float v = a.sums[(u * 2 + n) * a.cols + c];
        if (a.grad[n][0] != nullptr) {
          float other = 1.f;
          if (s.data != nullptr) other = (n ? 1.f : 0.f) + load_as_float(s.data, sample * s.pitch + c, s.dtype);
          total[n][0] = fmaf(v, other, total[n][0]);
        }
        total[n][1] += v;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) part[k][part_index][lane] = total[k >> 1][k & 1];
  __syncthreads();
  if (part_index < 4 && c < a.cols) {
    const int n = part_index >> 1, k = part_index & 1;
    const bool per_sample = a.factor[n][k].pitch != 0;
    if (a.grad[n][k] != nullptr && per_sample != shared_slot) {
      float sum = 0.f;
      for (int i = 0; i < 8; ++i) sum += part[part_index][i][lane];
      if (k == 1 && a.factor[n][0].data != nullptr)
        sum *= load_as_float(a.factor[n][0].data, c, a.factor[n][0].dtype);
      store_from_float(a.grad[n][k], per_sample ? (long long)blockIdx.x * a.cols + c : c, a.factor[n][k].dtype, sum);
    }
  }
}

}  // namespace vb

using namespace vb;

namespace {

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct NormShape {
  int vec, v, warps, groups;   // values per access, accesses per thread, warps per row, rows a block works on at a time
};

// Rows of 8-value pieces (16 bytes of a 16-bit type) where every row starts on a 16-byte boundary, single values else.
bool norm_shape(int cols, bool wide, NormShape& s) {
  if (cols < 1 || cols > VB_NORM_MAX_COLS || (wide && cols % 8)) return false;
  const int pieces = wide ? cols / 8 : cols;
  s.vec = wide ? 8 : 1;
  if (wide) s.v = pieces <= 256 ? 1 : pieces <= 1024 ? 2 : 4;
  else s.v = pieces <= 2048 ? 4 : 16;
  s.warps = (pieces + 32 * s.v - 1) / (32 * s.v);
  s.groups = s.warps == 1 ? 4 : 1;
  return true;
}

// blocks that fill the machine: about 1024 threads per SM
int norm_blocks(const NormShape& s) {
  const int threads = s.warps * s.groups * 32;
  return 148 * std::max(1, 1024 / threads);
}

template <typename TX, typename TY, int VEC, int V>
void launch_norm(const NormArgs& a, bool backward, bool post, bool pre, int blocks, int threads, cudaStream_t stream) {
  if (backward) {
    if (post && pre) norm_backward_kernel<TX, TY, VEC, V, true, true><<<blocks, threads, 0, stream>>>(a);
    else if (post) norm_backward_kernel<TX, TY, VEC, V, true, false><<<blocks, threads, 0, stream>>>(a);
    else norm_backward_kernel<TX, TY, VEC, V, false, true><<<blocks, threads, 0, stream>>>(a);
  } else {
    if (post && pre) norm_forward_kernel<TX, TY, VEC, V, true, true><<<blocks, threads, 0, stream>>>(a);
    else if (post) norm_forward_kernel<TX, TY, VEC, V, true, false><<<blocks, threads, 0, stream>>>(a);
    else norm_forward_kernel<TX, TY, VEC, V, false, true><<<blocks, threads, 0, stream>>>(a);
  }
}

template <typename TX, typename TY>
void launch_shape(const NormArgs& a, const NormShape& s, bool backward, bool post, bool pre, int blocks, cudaStream_t stream) {
  const int threads = s.warps * s.groups * 32;
  if (s.vec == 8) {
    if (s.v == 1) launch_norm<TX, TY, 8, 1>(a, backward, post, pre, blocks, threads, stream);
    else if (s.v == 2) launch_norm<TX, TY, 8, 2>(a, backward, post, pre, blocks, threads, stream);
    else launch_norm<TX, TY, 8, 4>(a, backward, post, pre, blocks, threads, stream);
  } else {
    if (s.v == 4) launch_norm<TX, TY, 1, 4>(a, backward, post, pre, blocks, threads, stream);
    else launch_norm<TX, TY, 1, 16>(a, backward, post, pre, blocks, threads, stream);
  }
}

int launch_types(const NormArgs& a, int x_dtype, int y_dtype, const NormShape& s, bool backward, bool post, bool pre,
                 int blocks, cudaStream_t stream) {
  if (x_dtype == kF32 && y_dtype == kF32) launch_shape<float, float>(a, s, backward, post, pre, blocks, stream);
  else if (x_dtype == kF32 && y_dtype == kBF16) launch_shape<float, __nv_bfloat16>(a, s, backward, post, pre, blocks, stream);
  else if (x_dtype == kF32 && y_dtype == kF16) launch_shape<float, __half>(a, s, backward, post, pre, blocks, stream);
  else if (x_dtype == kBF16 && y_dtype == kBF16) launch_shape<__nv_bfloat16, __nv_bfloat16>(a, s, backward, post, pre, blocks, stream);
  else if (x_dtype == kF16 && y_dtype == kF16) launch_shape<__half, __half>(a, s, backward, post, pre, blocks, stream);
  else return (int)cudaErrorInvalidValue;
  return (int)cudaGetLastError();
}

bool vector_ok(const VbNormVector& v, int cols) {
  return v.data == nullptr || (v.dtype >= kF32 && v.dtype <= kF16 && (v.pitch == 0 || v.pitch >= cols));
}
NormVector to_vector(const VbNormVector& v) { return NormVector{v.data, v.dtype, v.pitch}; }

// units of the backward pass: enough to fill the machine twice, at most one per row of a sample
int backward_units(const NormShape& s, int samples, int tokens) {
  const long long want = 2LL * norm_blocks(s) * s.groups;
  return (int)std::max<long long>(1, std::min<long long>(tokens, (want + samples - 1) / samples));
}
// the rule on pointers is the caller's: a workspace has to do for both
long long norm_workspace(int rows, int cols, int tokens, bool wide) {
  NormShape s;
  if (rows <= 0 || tokens <= 0 || rows % tokens || !norm_shape(cols, wide, s)) return 0;
  const int samples = rows / tokens;
  return (long long)samples * backward_units(s, samples, tokens) * 2 * cols;
}

}  // namespace

extern "C" long long vb_block_norm_workspace(int rows, int cols, int tokens) {
  return std::max(norm_workspace(rows, cols, tokens, true), norm_workspace(rows, cols, tokens, false));
}

extern "C" int vb_block_norm(const VbBlockNorm* n, cudaStream_t stream) {
  const bool post = n->y != nullptr, pre = n->h != nullptr;
  if (n->rows < 0 || n->tokens < 1 || n->rows % n->tokens || n->x == nullptr || (!post && !pre) || (post && n->out == nullptr) ||
      !vector_ok(n->weight, n->cols) || !vector_ok(n->gate, n->cols) || !vector_ok(n->next_weight, n->cols) ||
      !vector_ok(n->next_scale, n->cols))
    return (int)cudaErrorInvalidValue;
  NormShape s;
  const bool wide = n->cols % 8 == 0 && on16(n->x) && on16(n->y) && on16(n->out) && on16(n->h);
  if (!norm_shape(n->cols, wide, s)) return (int)cudaErrorInvalidValue;
  if (n->rows == 0) return 0;
  NormArgs a{};
  a.rows = n->rows; a.cols = n->cols; a.tokens = n->tokens; a.warps = s.warps;
  a.alpha = n->residual_scale; a.eps = n->eps;
  a.x = n->x; a.y = n->y;
  a.weight = to_vector(n->weight); a.gate = to_vector(n->gate);
  a.next_weight = to_vector(n->next_weight); a.next_scale = to_vector(n->next_scale);
  a.out = n->out; a.h = n->h; a.ry = n->ry; a.ru = n->ru;
  const int blocks = std::min((n->rows + s.groups - 1) / s.groups, norm_blocks(s));
  return launch_types(a, n->x_dtype, n->y_dtype, s, false, post, pre, blocks, stream);
}

extern "C" int vb_block_norm_backward(const VbBlockNorm* n, const VbBlockNormGrads* g, cudaStream_t stream) {
  const bool post = n->y != nullptr, pre = g->dh != nullptr;
  const bool post_sums = post && (g->dweight != nullptr || g->dgate != nullptr);
  const bool pre_sums = pre && (g->dnext_weight != nullptr || g->dnext_scale != nullptr);
  if (n->rows < 0 || n->tokens < 1 || n->rows % n->tokens || (!post && !pre) || (post && n->ry == nullptr) ||
      (pre && (n->ru == nullptr || n->x == nullptr)) || (!pre && g->dout == nullptr) || !vector_ok(n->weight, n->cols) ||
      !vector_ok(n->gate, n->cols) || !vector_ok(n->next_weight, n->cols) || !vector_ok(n->next_scale, n->cols))
    return (int)cudaErrorInvalidValue;
  NormShape s;
  const bool wide = n->cols % 8 == 0 && on16(n->x) && on16(n->y) && on16(g->dout) && on16(g->dh) && on16(g->dx) && on16(g->dy);
  if (!norm_shape(n->cols, wide, s)) return (int)cudaErrorInvalidValue;
  if (n->rows == 0) return 0;
  const int samples = n->rows / n->tokens, units = backward_units(s, samples, n->tokens);
  if ((post_sums || pre_sums) && (g->workspace == nullptr || g->workspace_floats < (long long)samples * units * 2 * n->cols))
    return (int)cudaErrorInvalidValue;
  NormArgs a{};
  a.rows = n->rows; a.cols = n->cols; a.tokens = n->tokens; a.warps = s.warps;
  a.alpha = n->residual_scale; a.eps = n->eps;
  a.x = n->x; a.y = n->y;
  a.weight = to_vector(n->weight); a.gate = to_vector(n->gate);
  a.next_weight = to_vector(n->next_weight); a.next_scale = to_vector(n->next_scale);
  a.ry = n->ry; a.ru = n->ru;
  a.dout = g->dout; a.dh = g->dh; a.dx = g->dx; a.dy = g->dy;
  a.units_per_sample = units;
  a.sums = post_sums || pre_sums ? g->workspace : nullptr;
  const long long blocks = ((long long)samples * units + s.groups - 1) / s.groups;
  if (blocks > INT_MAX) return (int)cudaErrorInvalidValue;
  const int rc = launch_types(a, n->x_dtype, n->y_dtype, s, true, post, pre, (int)blocks, stream);
  if (rc != 0 || a.sums == nullptr) return rc;
  NormSumArgs t{};
  t.cols = n->cols; t.samples = samples; t.units_per_sample = units; t.sums = g->workspace;
  t.factor[0][0] = a.weight; t.factor[0][1] = a.gate;
  t.factor[1][0] = a.next_weight; t.factor[1][1] = a.next_scale;
  if (post) { t.grad[0][0] = g->dweight; t.grad[0][1] = g->dgate; }
  if (pre) { t.grad[1][0] = g->dnext_weight; t.grad[1][1] = g->dnext_scale; }
  norm_sums_kernel<<<dim3(samples + 1, (n->cols + 31) / 32), 256, 0, stream>>>(t);
  return (int)cudaGetLastError();
}
