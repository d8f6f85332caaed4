// RMS norms after and before a transformer block, fused with the block's gate and the residual scale:
//
//   yh  = y * ry,  ry = (mean(y^2) + eps)^-1/2              (POST: the norm after the block)
//   u   = alpha * x + gate * weight * yh                    -> out, the residual stream
//   h   = u * ru * next_weight * (1 + next_scale)           (PRE: the norm before the next block; u = x without POST)
//
// One pass each way: a row's values stay in registers between the statistics and the results, and the backward pass
// forms u again from x and y, which the graph holds anyway, so nothing but the two reciprocal roots is saved.
// Vectors are fp32, bf16 or fp16 with a pitch per sample (0: one vector for all rows); all arithmetic is fp32.
#include <atomic>
#include <climits>

#include "api.h"
#include "common/numerics.cuh"

namespace vb {

constexpr unsigned kAll = 0xffffffffu;

struct NormVector {            // [samples, cols] (or [cols] with pitch 0), null = absent
  const void* data;
  int dtype;
  int wide;                    // rows start on 16-byte boundaries
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
  void *dgate, *dnext_scale;   // gradients of per-sample vectors, or null
  float* sums;                 // [blocks][2][cols]: column sums of d * yh and of dh * uh for the shared vectors, or null
  float* parked;               // [row groups][2][2][cols]: the same of samples that another group shares, or null
  int depth;                   // rows fetched ahead (0: none)
  int slot_bytes;              // shared memory of one fetched row
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

// ---- fetching rows ahead -------------------------------------------------------------------------------------------
// A thread copies the pieces of the next rows that it will need itself into its own 16-byte places in shared memory
// (cp.async), so nothing but its own copies has to be waited for: no barrier, and no registers hold the rows in flight.
__device__ __forceinline__ void copy_ahead(uint32_t to, const void* from, bool through_l1) {
  if (through_l1) asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copy_wait(int pending) {     // all but the youngest `pending` groups have arrived
  if (pending >= 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
  else if (pending == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 1;" ::: "memory");
}

// One tensor's part of a slot: V pieces of VEC values per thread, 16-byte words of neighbouring threads next to each other
template <typename T, int VEC, int V> struct Strip {
  static constexpr int kWords = Piece<T, VEC>::kBytes / 16;  // 0: too narrow to be fetched ahead
  __device__ __forceinline__ static int bytes(int threads) { return V * kWords * threads * 16; }
  // fp32 pieces are two words apart in memory: the halves of a 32-byte sector meet in L1
  __device__ __forceinline__ static void fetch(uint32_t slot, const T* row, int tid, int threads, int cols) {
    if constexpr (kWords > 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = (tid + j * threads) * VEC;
        if (c < cols)
#pragma unroll
          for (int w = 0; w < kWords; ++w)
            copy_ahead(slot + ((j * kWords + w) * threads + tid) * 16, row + c + w * (16 / (int)sizeof(T)), kWords > 1);
      }
    }
  }
  __device__ __forceinline__ static void take(const unsigned char* slot, int j, int tid, int threads, Piece<T, VEC>& piece) {
    if constexpr (kWords > 0) {
#pragma unroll
      for (int w = 0; w < kWords; ++w)
        piece.word[w] = *reinterpret_cast<const uint4*>(slot + ((j * kWords + w) * threads + tid) * 16);
    }
  }
};

// Sums N values over the warps of a row; every thread gets them.  `turn` alternates between two buffers, so that one
// barrier per call is enough: a warp can only reach the buffer's next use through the other buffer's barrier.
// Rows that a block works on at the same time meet at barriers of their own.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int warps, int group, float (*buffer)[N][32], int& turn) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[n] += __shfl_xor_sync(kAll, v[n], o);
  if (warps == 1) return;
  const int lane = threadIdx.x & 31, first = group * warps;
  if (lane == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) buffer[turn][n][threadIdx.x >> 5] = v[n];
  }
  // (named one by one: a barrier number in a register would reserve all sixteen for the block)
  if (group == 0) asm volatile("bar.sync 1, %0;" ::"r"(warps * 32) : "memory");
  else if (group == 1) asm volatile("bar.sync 2, %0;" ::"r"(warps * 32) : "memory");
  else if (group == 2) asm volatile("bar.sync 3, %0;" ::"r"(warps * 32) : "memory");
  else asm volatile("bar.sync 4, %0;" ::"r"(warps * 32) : "memory");
  if (warps <= 4) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = buffer[turn][n][first] + buffer[turn][n][first + 1];
      if (warps > 2) v[n] += buffer[turn][n][first + 2];
      if (warps > 3) v[n] += buffer[turn][n][first + 3];
    }
  } else {
    // every warp adds the warps' sums for itself: one value a lane, 8, 16 or 32 lanes
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = lane < warps ? buffer[turn][n][first + lane] : 0.f;
    if (warps > 16)
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(kAll, v[n], 16);
    if (warps > 8)
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(kAll, v[n], 8);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1)
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(kAll, v[n], o);
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = __shfl_sync(kAll, v[n], 0);
  }
  turn ^= 1;
}

// fp32 values of a thread's columns in shared memory, in places of its own (no barrier): value i of piece j
template <int VEC>
__device__ __forceinline__ int own_place(int j, int i, int tid, int threads) {
  return VEC == 1 ? j * threads + tid : ((j * (VEC / 4) + i / 4) * threads + tid) * 4 + i % 4;
}
template <int VEC>
__device__ __forceinline__ void own_values(const float* area, int j, int tid, int threads, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = area[own_place<VEC>(j, 0, tid, threads)];
  } else {
#pragma unroll
    for (int w = 0; w < VEC / 4; ++w) {
      const float4 f = *reinterpret_cast<const float4*>(area + own_place<VEC>(j, 4 * w, tid, threads));
      v[4 * w] = f.x; v[4 * w + 1] = f.y; v[4 * w + 2] = f.z; v[4 * w + 3] = f.w;
    }
  }
}

__device__ __forceinline__ float vector_value(const NormVector& v, long long sample, int c, float shift, float otherwise) {
  return v.data != nullptr ? shift + load_as_float(v.data, sample * v.pitch + c, v.dtype) : otherwise;
}
// VEC neighbouring values of an optional vector (absent: 1) plus `shift`
template <int VEC>
__device__ __forceinline__ void vector_values(const NormVector& v, long long sample, int c, float shift, float (&f)[VEC]) {
  if (v.data == nullptr) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = 1.f;
    return;
  }
  const long long at = sample * v.pitch + c;
  if (VEC == 8 && v.wide) {
    if (v.dtype == kF32) {
      const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(v.data) + at);
#pragma unroll
      for (int w = 0; w < VEC / 4; ++w) {
        const float4 t = p[w];
        f[4 * w] = t.x; f[4 * w + 1] = t.y; f[4 * w + 2] = t.z; f[4 * w + 3] = t.w;
      }
    } else {
      Piece<__nv_bfloat16, VEC> raw;
      raw.load(reinterpret_cast<const __nv_bfloat16*>(v.data) + at);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        f[i] = v.dtype == kBF16 ? raw.get(i) : __half2float(__ushort_as_half(__bfloat16_as_ushort(raw.value[i])));
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = load_as_float(v.data, at + i, v.dtype);
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] += shift;
}

// product of two optional vectors (the second plus `shift`) for the columns of one thread; once per sample
template <int VEC, int V>
__device__ __forceinline__ void store_gain(const NormVector& a, const NormVector& b, float shift, long long sample, int tid,
                                           int threads, int cols, float* area) {
#pragma unroll 1
  for (int j = 0; j < V; ++j) {
    const int c = (tid + j * threads) * VEC;
    if (c < cols) {
      float f[VEC], g[VEC];
      vector_values<VEC>(a, sample, c, 0.f, f);
      vector_values<VEC>(b, sample, c, shift, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) area[own_place<VEC>(j, i, tid, threads)] = f[i] * g[i];
    }
  }
}

// pieces of rows too wide for registers are walked without unrolling
#define VB_PIECES _Pragma("unroll (V > 4 ? 1 : V)")

template <typename TX, typename TY, int VEC, int V, bool POST, bool PRE>
__global__ void __launch_bounds__(VEC == 1 ? 1024 : 512)
norm_forward_kernel(const NormArgs a) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float buffer[2][1][32];
  using SX = Strip<TX, VEC, V>;
  using SY = Strip<TY, VEC, V>;
  const int threads = a.warps * 32, group = threadIdx.x / threads, tid = threadIdx.x - group * threads;
  const int groups = blockDim.x / threads, units = gridDim.x * groups;
  const int per_unit = (a.rows + units - 1) / units;
  const long long first = (long long)(blockIdx.x * groups + group) * per_unit;
  const long long last = min(first + per_unit, (long long)a.rows);
  const TX* x = reinterpret_cast<const TX*>(a.x);
  const TY* y = reinterpret_cast<const TY*>(a.y);
  const float inverse = 1.f / (float)a.cols;
  const int slots = a.depth + 1, x_bytes = SX::bytes(threads);
  unsigned char* mine = ring + (size_t)group * slots * a.slot_bytes;
  auto fetch = [&](long long row, int place) {
    if (row < last) {
      const uint32_t slot = (uint32_t)__cvta_generic_to_shared(mine + place * a.slot_bytes);
      SX::fetch(slot, x + row * a.cols, tid, threads, a.cols);
      if (POST) SY::fetch(slot + x_bytes, y + row * a.cols, tid, threads, a.cols);
    }
    copy_commit();
  };
  for (int d = 0; d < a.depth; ++d) fetch(first + d, d);
  float* gains = reinterpret_cast<float*>(ring + (size_t)groups * slots * a.slot_bytes) + (size_t)group * 2 * V * VEC * threads;
  float* next_gains = gains + V * VEC * threads;
  long long sample = first / a.tokens, sample_end = first;
  int turn = 0, head = 0;
  for (long long row = first; row < last; ++row) {
    Piece<TX, VEC> px[V];
    Piece<TY, VEC> py[V];
    const long long base = row * a.cols;
    if (VEC > 1 && a.depth > 0) {
      const int ahead = head + a.depth;
      fetch(row + a.depth, ahead >= slots ? ahead - slots : ahead);
      copy_wait(a.depth);
      const unsigned char* slot = mine + head * a.slot_bytes;
      head = head + 1 == slots ? 0 : head + 1;
VB_PIECES
      for (int j = 0; j < V; ++j) {
        SX::take(slot, j, tid, threads, px[j]);
        if (POST) SY::take(slot + x_bytes, j, tid, threads, py[j]);
      }
    } else {
VB_PIECES
      for (int j = 0; j < V; ++j) {
        const int c = (tid + j * threads) * VEC;
        if (c < a.cols) {
          px[j].load(x + base + c);
          if (POST) py[j].load(y + base + c);
        }
      }
    }
    if (row >= sample_end) {
      if (row > first) ++sample;
      sample_end = (sample + 1) * a.tokens;
      if (POST) store_gain<VEC, V>(a.weight, a.gate, 0.f, sample, tid, threads, a.cols, gains);
      if (PRE) store_gain<VEC, V>(a.next_weight, a.next_scale, 1.f, sample, tid, threads, a.cols, next_gains);
    }
    float u[V][VEC], sum[1] = {0.f};
    if (POST) {
VB_PIECES
      for (int j = 0; j < V; ++j)
        if ((tid + j * threads) * VEC < a.cols)
#pragma unroll
          for (int i = 0; i < VEC; ++i) sum[0] = fmaf(py[j].get(i), py[j].get(i), sum[0]);
      row_sum<1>(sum, a.warps, group, buffer, turn);
      const float ry = rsqrtf(fmaf(sum[0], inverse, a.eps));
      if (tid == 0 && a.ry != nullptr) a.ry[row] = ry;
VB_PIECES
      for (int j = 0; j < V; ++j) {
        const int c = (tid + j * threads) * VEC;
        if (c < a.cols) {
          Piece<TX, VEC> o;
          float gain[VEC];
          own_values<VEC>(gains, j, tid, threads, gain);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            u[j][i] = fmaf(a.alpha, px[j].get(i), py[j].get(i) * ry * gain[i]);
            o.set(i, u[j][i]);
          }
          o.store(reinterpret_cast<TX*>(a.out) + base + c);
        }
      }
    } else {
VB_PIECES
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) u[j][i] = px[j].get(i);
    }
    if (PRE) {
      sum[0] = 0.f;
VB_PIECES
      for (int j = 0; j < V; ++j)
        if ((tid + j * threads) * VEC < a.cols)
#pragma unroll
          for (int i = 0; i < VEC; ++i) sum[0] = fmaf(u[j][i], u[j][i], sum[0]);
      row_sum<1>(sum, a.warps, group, buffer, turn);
      const float ru = rsqrtf(fmaf(sum[0], inverse, a.eps));
      if (tid == 0 && a.ru != nullptr) a.ru[row] = ru;
VB_PIECES
      for (int j = 0; j < V; ++j) {
        const int c = (tid + j * threads) * VEC;
        if (c < a.cols) {
          Piece<TY, VEC> o;
          float gain[VEC];
          own_values<VEC>(next_gains, j, tid, threads, gain);
#pragma unroll
          for (int i = 0; i < VEC; ++i) o.set(i, u[j][i] * ru * gain[i]);
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
//
// Column sums S = sum of d * yh and R = sum of dh * uh give the gradients of the vectors.  Every row group (a block, or
// part of one where rows are short) takes an equal share of consecutive rows.  SAMPLES: at the end of a sample it writes
// the gradients of the per-sample vectors if it had the whole sample, else parks the sums (place 0: the sample began in
// an earlier group, 1: it goes on in a later one), and adds them, weighted with the per-sample partner, to the sums of
// the shared vectors.
template <typename TX, typename TY, int VEC, int V, bool POST, bool PRE, bool SAMPLES>
__global__ void __launch_bounds__(VEC == 1 ? 1024 : 512)
norm_backward_kernel(const NormArgs a) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float buffer[2][3][32];
  using SX = Strip<TX, VEC, V>;
  using SY = Strip<TY, VEC, V>;
  const int threads = a.warps * 32, group = threadIdx.x / threads, tid = threadIdx.x - group * threads;
  const int groups = blockDim.x / threads;
  const TX* x = reinterpret_cast<const TX*>(a.x);
  const TY* y = reinterpret_cast<const TY*>(a.y);
  const TX* dout = reinterpret_cast<const TX*>(a.dout);
  const TY* dh = reinterpret_cast<const TY*>(a.dh);
  const float inverse = 1.f / (float)a.cols;
  const long long unit = (long long)blockIdx.x * groups + group, units = min((long long)gridDim.x * groups, (long long)a.rows);
  const long long first = a.rows * min(unit, units) / units, last = a.rows * min(unit + 1, units) / units;
  const int slots = a.depth + 1, x_bytes = SX::bytes(threads), y_bytes = SY::bytes(threads);
  unsigned char* mine = ring + (size_t)group * slots * a.slot_bytes;
  // dout and, for PRE, x; y for POST; dh for PRE
  const int at_dout = PRE ? x_bytes : 0, at_y = at_dout + (a.dout != nullptr ? x_bytes : 0), at_dh = at_y + (POST ? y_bytes : 0);
  int head = 0;
  auto fetch = [&](long long row, int place) {
    if (row < last) {
      const uint32_t slot = (uint32_t)__cvta_generic_to_shared(mine + place * a.slot_bytes);
      const long long base = row * a.cols;
      if (PRE) SX::fetch(slot, x + base, tid, threads, a.cols);
      if (a.dout != nullptr) SX::fetch(slot + at_dout, dout + base, tid, threads, a.cols);
      if (POST) SY::fetch(slot + at_y, y + base, tid, threads, a.cols);
      if (PRE) SY::fetch(slot + at_dh, dh + base, tid, threads, a.cols);
    }
    copy_commit();
  };
  for (int d = 0; d < a.depth; ++d) fetch(first + d, d);

  float post_sum[V][VEC], pre_sum[V][VEC];
VB_PIECES
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int i = 0; i < VEC; ++i) post_sum[j][i] = pre_sum[j][i] = 0.f;
  // per group: gains, next gains; then, where sums of several samples or groups meet, sums of S and R
  const int area = V * VEC * threads;
  float* gains = reinterpret_cast<float*>(ring + (size_t)groups * slots * a.slot_bytes) + (size_t)group * 2 * area;
  float* next_gains = gains + area;
  float* total = reinterpret_cast<float*>(ring + (size_t)groups * slots * a.slot_bytes) + (size_t)(groups + group) * 2 * area;
  constexpr bool kTotalsShared = V * VEC <= 8;  // wider rows (one group to a block) keep the sums in their final place
  if (SAMPLES && kTotalsShared) {
#pragma unroll 1
    for (int k = 0; k < 2 * V * VEC; ++k) total[k * threads + tid] = 0.f;
  }
  const long long first_sample = SAMPLES ? first / a.tokens : 0;
  auto finish_norm = [&](int n, long long sample, const NormVector& weight, const NormVector& partner, float shift, void* grad,
                         float (&sum)[V][VEC]) {
    const bool fresh = sample == first_sample, before = sample * a.tokens < first, after = (sample + 1) * a.tokens > last;
    float* park = a.parked + ((unit * 2 + (before ? 0 : 1)) * 2 + n) * a.cols;
VB_PIECES
    for (int j = 0; j < V; ++j) {
      const int c = (tid + j * threads) * VEC;
      if (c < a.cols) {
        float f[VEC];
        if (grad != nullptr) {
          if (before || after) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) park[c + i] = sum[j][i];
          } else {
            vector_values<VEC>(weight, 0, c, 0.f, f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) store_from_float(grad, sample * a.cols + c + i, partner.dtype, sum[j][i] * f[i]);
          }
        }
        if (a.sums != nullptr) {
          if (partner.pitch != 0) {
            vector_values<VEC>(partner, sample, c, shift, f);
          } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = 1.f;
          }
          if constexpr (kTotalsShared) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) total[n * area + own_place<VEC>(j, i, tid, threads)] += sum[j][i] * f[i];
          } else {
            float* to = a.sums + ((long long)blockIdx.x * 2 + n) * a.cols + c;
#pragma unroll
            for (int i = 0; i < VEC; ++i) to[i] = (fresh ? 0.f : to[i]) + sum[j][i] * f[i];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum[j][i] = 0.f;
    }
  };
  auto finish_sample = [&](long long sample) {
    if (POST) finish_norm(0, sample, a.weight, a.gate, 0.f, a.dgate, post_sum);
    if (PRE) finish_norm(1, sample, a.next_weight, a.next_scale, 1.f, a.dnext_scale, pre_sum);
  };

  long long sample = first_sample, sample_end = first;
  int turn = 0;
  for (long long row = first; row < last; ++row) {
    const long long base = row * a.cols;
    const float ry = POST ? a.ry[row] : 0.f, ru = PRE ? a.ru[row] : 0.f;
    if (row >= sample_end) {
      if (SAMPLES && row > first) finish_sample(sample++);
      sample_end = SAMPLES ? (sample + 1) * a.tokens : last;
      if (POST) store_gain<VEC, V>(a.weight, a.gate, 0.f, sample, tid, threads, a.cols, gains);
      if (PRE) store_gain<VEC, V>(a.next_weight, a.next_scale, 1.f, sample, tid, threads, a.cols, next_gains);
    }
    const unsigned char* slot = mine + head * a.slot_bytes;
    if (VEC > 1 && a.depth > 0) {
      const int ahead = head + a.depth;
      fetch(row + a.depth, ahead >= slots ? ahead - slots : ahead);
      copy_wait(a.depth);
      head = head + 1 == slots ? 0 : head + 1;
    }
    float d[V][VEC], yh[V][VEC], uh[V][VEC], sum[3] = {0.f, 0.f, 0.f};
VB_PIECES
    for (int j = 0; j < V; ++j) {
      const int c = (tid + j * threads) * VEC;
      Piece<TX, VEC> px, pd;
      Piece<TY, VEC> py, ph;
      float gain[VEC], next_gain[VEC];
      if (c < a.cols) {
        if (POST) own_values<VEC>(gains, j, tid, threads, gain);
        if (PRE) own_values<VEC>(next_gains, j, tid, threads, next_gain);
        if (VEC > 1 && a.depth > 0) {
          if (PRE) SX::take(slot, j, tid, threads, px);
          if (a.dout != nullptr) SX::take(slot + at_dout, j, tid, threads, pd);
          if (POST) SY::take(slot + at_y, j, tid, threads, py);
          if (PRE) SY::take(slot + at_dh, j, tid, threads, ph);
        } else {
          if (PRE) px.load(x + base + c);
          if (POST) py.load(y + base + c);
          if (a.dout != nullptr) pd.load(dout + base + c);
          if (PRE) ph.load(dh + base + c);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float q = 0.f, u;
          d[j][i] = a.dout != nullptr ? pd.get(i) : 0.f;
          if (POST) {
            yh[j][i] = py.get(i) * ry;
            q = yh[j][i] * gain[i];
          }
          if (PRE) {
            u = POST ? fmaf(a.alpha, px.get(i), q) : px.get(i);
            uh[j][i] = u * ru;
            const float g = ph.get(i), t = g * next_gain[i];
            pre_sum[j][i] = fmaf(g, uh[j][i], pre_sum[j][i]);
            sum[0] = fmaf(t, uh[j][i], sum[0]);
            d[j][i] = fmaf(ru, t, d[j][i]);
            if (POST) sum[2] = fmaf(uh[j][i], q, sum[2]);
          }
          if (POST) sum[1] = fmaf(d[j][i], q, sum[1]);
        }
      }
    }
    row_sum<3>(sum, a.warps, group, buffer, turn);
    const float pull = ru * sum[0] * inverse;                       // ru c
    const float m = POST ? (PRE ? fmaf(-pull, sum[2], sum[1]) : sum[1]) * inverse : 0.f;
VB_PIECES
    for (int j = 0; j < V; ++j) {
      const int c = (tid + j * threads) * VEC;
      if (c < a.cols) {
        Piece<TX, VEC> ox;
        Piece<TY, VEC> oy;
        float gain[VEC];
        if (POST) own_values<VEC>(gains, j, tid, threads, gain);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float whole = PRE ? fmaf(-pull, uh[j][i], d[j][i]) : d[j][i];
          ox.set(i, POST ? a.alpha * whole : whole);
          if (POST) {
            oy.set(i, ry * fmaf(-m, yh[j][i], whole * gain[i]));
            post_sum[j][i] = fmaf(whole, yh[j][i], post_sum[j][i]);
          }
        }
        if (a.dx != nullptr) ox.store(reinterpret_cast<TX*>(a.dx) + base + c);
        if (POST && a.dy != nullptr) oy.store(reinterpret_cast<TY*>(a.dy) + base + c);
      }
    }
  }
  if (SAMPLES && first < last) finish_sample(sample);
  if (a.sums == nullptr || (SAMPLES && !kTotalsShared)) return;
  float* to = a.sums + (long long)blockIdx.x * 2 * a.cols;
  if (!SAMPLES && groups == 1) {
VB_PIECES
    for (int j = 0; j < V; ++j) {
      const int c = (tid + j * threads) * VEC;
      if (c < a.cols)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          to[c + i] = POST ? post_sum[j][i] : 0.f;
          to[a.cols + c + i] = PRE ? pre_sum[j][i] : 0.f;
        }
    }
    return;
  }
  if (!SAMPLES) {
VB_PIECES
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        total[own_place<VEC>(j, i, tid, threads)] = POST ? post_sum[j][i] : 0.f;
        total[area + own_place<VEC>(j, i, tid, threads)] = PRE ? pre_sum[j][i] : 0.f;
      }
  }
  __syncthreads();
  // the first group adds the groups' sums in order
  if (group == 0) {
#pragma unroll 1
    for (int k = 0; k < 2 * V * VEC; ++k) {
      const int n = k / (V * VEC), j = k / VEC % V, i = k % VEC, c = (tid + j * threads) * VEC + i;
      if (c < a.cols) {
        const float* from = total + n * area + own_place<VEC>(j, i, tid, threads);
        float s = from[0];
        for (int g = 1; g < groups; ++g) s += from[(size_t)g * 2 * area];
        to[n * a.cols + c] = s;
      }
    }
  }
}

struct NormSumArgs {
  int rows, cols, tokens;
  int blocks;                  // sets of sums, 0 if nothing is shared
  long long units;             // row groups of the backward kernel that have rows
  const float *sums, *parked;
  NormVector weight[2], partner[2];          // of the two norms: weight, and gate / next_scale
  void *dweight[2], *dpartner[2];            // gradients, or null
};

// Gradients of the vectors from what the row groups left.  The shared ones: with T the sum of the blocks' sums, T for a
// weight whose partner is per sample (its factors are in T), partner * T for one whose partner is shared, and weight * T
// for a shared partner.  Per-sample ones of samples that several groups shared: weight * sum of what they parked.
// A block has 128 columns, 4 a thread, and 32 rows of threads: the first block of a column range (where anything is
// shared) gives all of them to T, every other one eight to each of four group boundaries; the first boundary inside a
// sample takes that sample.  A row takes every 32nd (8th) set, and the rows are added in order.
__global__ void __launch_bounds__(1024)
norm_sums_kernel(const NormSumArgs a) {
  __shared__ float4 part[2][32][32];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, c = blockIdx.y * 128 + lane * 4;
  const int has_shared = a.blocks > 0 ? 1 : 0;
  const bool shared_block = has_shared && blockIdx.x == 0;
  const int stride = shared_block ? 32 : 8, turn = shared_block ? row : row % 8;
  const float* from = a.sums;
  long long sample = 0, first = 0, last = a.blocks;
  if (!shared_block) {
    from = a.parked;
    first = last = 0;
    const long long unit = ((long long)blockIdx.x - has_shared) * 4 + row / 8 + 1;
    if (unit < a.units) {
      const long long begin = a.rows * unit / a.units;
      sample = begin / a.tokens;
      const long long start = sample * a.tokens;
      if (begin > start && begin < a.rows && a.rows * (unit - 1) / a.units <= start) {
        first = unit - 1;
        last = ((start + a.tokens) * a.units - 1) / a.rows + 1;     // behind the group that has the sample's last row
      }
    }
  }
  bool wanted[2];                               // the same for the whole block
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const bool per_sample = a.partner[n].pitch != 0;
    wanted[n] = shared_block ? a.dweight[n] != nullptr || (a.dpartner[n] != nullptr && !per_sample)
                             : a.dpartner[n] != nullptr && per_sample;
  }
  float total[2][4] = {};
#pragma unroll 4
  for (long long u = first + turn; u < last; u += stride) {
    const long long set = shared_block ? u : u * 2 + (u > first ? 0 : 1);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if (!wanted[n] || c >= a.cols) continue;
      const float* at = from + (set * 2 + n) * a.cols + c;
      if (a.cols % 4 == 0) {
        const float4 t = *reinterpret_cast<const float4*>(at);
        total[n][0] += t.x; total[n][1] += t.y; total[n][2] += t.z; total[n][3] += t.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c + i < a.cols) total[n][i] += at[i];
      }
    }
  }
#pragma unroll
  for (int n = 0; n < 2; ++n) part[n][row][lane] = make_float4(total[n][0], total[n][1], total[n][2], total[n][3]);
  __syncthreads();
  // rows 0 and 1 of a set (four sets of eight, or one) finish one norm each
  const int n = turn;
  if (turn >= 2 || first >= last || !wanted[n]) return;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = row - turn; i < row - turn + stride; ++i) {
    const float4 t = part[n][i][lane];
    sum[0] += t.x; sum[1] += t.y; sum[2] += t.z; sum[3] += t.w;
  }
  const NormVector &w = a.weight[n], &p = a.partner[n];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (c + i >= a.cols) continue;
    const float by_weight = sum[i] * vector_value(w, 0, c + i, 0.f, 1.f);
    if (!shared_block) {
      store_from_float(a.dpartner[n], sample * a.cols + c + i, p.dtype, by_weight);
    } else {
      if (a.dweight[n] != nullptr)
        store_from_float(a.dweight[n], c + i, w.dtype, p.pitch != 0 ? sum[i] : sum[i] * vector_value(p, 0, c + i, n ? 1.f : 0.f, 1.f));
      if (a.dpartner[n] != nullptr && p.pitch == 0) store_from_float(a.dpartner[n], c + i, p.dtype, by_weight);
    }
  }
}

}  // namespace vb

using namespace vb;

namespace {

constexpr int kSharedPerBlock = 227 * 1024;
constexpr int kBackwardThreads = 512;        // that an SM's registers do for

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct NormShape {
  int vec, v, warps, groups;   // values per access, accesses per thread, warps per row, rows a block works on at a time
  int threads() const { return warps * groups * 32; }
};

// Rows of 8-value pieces (16 bytes of a 16-bit type) where every row starts on a 16-byte boundary, single values else.
bool norm_shape(int cols, bool wide, NormShape& s) {
  if (cols < 1 || cols > VB_NORM_MAX_COLS || (wide && cols % 8)) return false;
  const int pieces = wide ? cols / 8 : cols;
  s.vec = wide ? 8 : 1;
  if (wide) s.v = pieces <= 512 ? 1 : pieces <= 1024 ? 2 : 4;
  else s.v = pieces <= 2048 ? 4 : 16;
  s.warps = (pieces + 32 * s.v - 1) / (32 * s.v);
  s.groups = std::max(1, 8 / s.warps);
  return true;
}

// Rows fetched ahead (as many up to three as cost no resident block), shared memory for them and for `areas` fp32 values
// per column, and blocks that one SM holds where its registers do for `resident_threads`.
struct NormPlan {
  int depth, slot_bytes, resident;
  size_t smem;
};
int by_registers(const NormShape& s, int resident_threads) { return std::max(1, resident_threads / s.threads()); }
NormPlan norm_plan(const NormShape& s, int row_bytes_per_value, int areas, int resident_threads) {
  NormPlan p{0, 0, 1, 0};
  const size_t extra = (size_t)areas * s.v * s.vec * s.threads() * sizeof(float);
  const int most = by_registers(s, resident_threads);
  const int slot = s.vec == 8 ? s.v * s.warps * 32 * 8 * row_bytes_per_value : 0;
  for (p.depth = slot ? 3 : 0;; --p.depth) {
    p.smem = extra + (p.depth ? (size_t)(p.depth + 1) * s.groups * slot : 0);
    p.resident = std::min(most, (int)(kSharedPerBlock / (p.smem + 2048)));
    if (p.resident == most || p.depth == 0 || (p.depth == 1 && p.resident > 0)) break;
  }
  p.slot_bytes = p.depth ? slot : 0;
  return p;
}

// lets a kernel use as much dynamic shared memory as its launch asks for, once per device
template <auto Kernel>
void allow_shared() {
  static std::atomic<unsigned long long> done{0};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return;
  const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
  if (bit && (done.load(std::memory_order_relaxed) & bit)) return;
  // what the kernel has statically comes off the limit: two row-sum buffers
  cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedPerBlock - 1024);
  done.fetch_or(bit, std::memory_order_relaxed);
}

struct NormLaunch {
  bool backward, post, pre, samples;
  int blocks, threads;
  size_t smem;
  cudaStream_t stream;
};

template <auto Kernel>
void launch_kernel(const NormArgs& a, const NormLaunch& l) {
  if (l.smem > 48 * 1024 - 1024) allow_shared<Kernel>();
  Kernel<<<l.blocks, l.threads, l.smem, l.stream>>>(a);
}

template <typename TX, typename TY, int VEC, int V, bool POST, bool PRE>
void launch_parts(const NormArgs& a, const NormLaunch& l) {
  if (!l.backward) launch_kernel<norm_forward_kernel<TX, TY, VEC, V, POST, PRE>>(a, l);
  else if (l.samples) launch_kernel<norm_backward_kernel<TX, TY, VEC, V, POST, PRE, true>>(a, l);
  else launch_kernel<norm_backward_kernel<TX, TY, VEC, V, POST, PRE, false>>(a, l);
}

template <typename TX, typename TY, int VEC, int V>
void launch_norms(const NormArgs& a, const NormLaunch& l) {
  if (l.post && l.pre) launch_parts<TX, TY, VEC, V, true, true>(a, l);
  else if (l.post) launch_parts<TX, TY, VEC, V, true, false>(a, l);
  else launch_parts<TX, TY, VEC, V, false, true>(a, l);
}

template <typename TX, typename TY>
void launch_shape(const NormArgs& a, const NormShape& s, const NormLaunch& l) {
  if (s.vec == 8) {
    if (s.v == 1) launch_norms<TX, TY, 8, 1>(a, l);
    else if (s.v == 2) launch_norms<TX, TY, 8, 2>(a, l);
    else launch_norms<TX, TY, 8, 4>(a, l);
  } else {
    if (s.v == 4) launch_norms<TX, TY, 1, 4>(a, l);
    else launch_norms<TX, TY, 1, 16>(a, l);
  }
}

int launch_types(const NormArgs& a, int x_dtype, int y_dtype, const NormShape& s, const NormLaunch& l) {
  if (x_dtype == kF32 && y_dtype == kF32) launch_shape<float, float>(a, s, l);
  else if (x_dtype == kF32 && y_dtype == kBF16) launch_shape<float, __nv_bfloat16>(a, s, l);
  else if (x_dtype == kF32 && y_dtype == kF16) launch_shape<float, __half>(a, s, l);
  else if (x_dtype == kBF16 && y_dtype == kBF16) launch_shape<__nv_bfloat16, __nv_bfloat16>(a, s, l);
  else if (x_dtype == kF16 && y_dtype == kF16) launch_shape<__half, __half>(a, s, l);
  else return (int)cudaErrorInvalidValue;
  return (int)cudaGetLastError();
}

bool vector_ok(const VbNormVector& v, int cols) {
  return v.data == nullptr || (v.dtype >= kF32 && v.dtype <= kF16 && (v.pitch == 0 || v.pitch >= cols));
}
int dtype_size(int dtype) { return dtype == kF32 ? 4 : 2; }
NormVector to_vector(const VbNormVector& v) {
  return NormVector{v.data, v.dtype, on16(v.data) && v.pitch * dtype_size(v.dtype) % 16 == 0, v.pitch};
}

// Blocks and shared memory of the backward pass: one wave, at least one row to a group
bool backward_plan(int rows, int cols, int tokens, int x_values, int y_values, bool wide, NormShape& s, NormPlan& p, int& blocks) {
  if (!norm_shape(cols, wide, s)) return false;
  p = norm_plan(s, x_values + y_values, s.v * s.vec <= 8 && (tokens < rows || s.groups > 1) ? 4 : 2, kBackwardThreads);
  blocks = std::min((rows + s.groups - 1) / s.groups, 148 * p.resident);
  return true;
}
// sums of the shared vectors, and, with samples, what groups park
long long backward_floats(const NormShape& s, int blocks, int rows, int cols, int tokens) {
  return (long long)blocks * 2 * cols * (1 + (tokens < rows ? 2 * s.groups : 0));
}

}  // namespace

// the most that any types and pointers lead to
extern "C" long long vb_block_norm_workspace(int rows, int cols, int tokens) {
  if (rows <= 0 || cols <= 0 || tokens <= 0 || rows % tokens || cols > VB_NORM_MAX_COLS) return 0;
  long long floats = 0;
  for (const bool wide : {true, false}) {
    NormShape s;
    if (!norm_shape(cols, wide, s)) continue;
    const int blocks = std::min((rows + s.groups - 1) / s.groups, 148 * by_registers(s, kBackwardThreads));
    floats = std::max(floats, backward_floats(s, blocks, rows, cols, tokens));
  }
  return floats;
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
  const NormPlan p = norm_plan(s, dtype_size(n->x_dtype) + (post ? dtype_size(n->y_dtype) : 0), 2, s.v * s.vec <= 8 ? 1024 : 512);
  NormArgs a{};
  a.rows = n->rows; a.cols = n->cols; a.tokens = n->tokens; a.warps = s.warps;
  a.alpha = n->residual_scale; a.eps = n->eps;
  a.x = n->x; a.y = n->y;
  a.weight = to_vector(n->weight); a.gate = to_vector(n->gate);
  a.next_weight = to_vector(n->next_weight); a.next_scale = to_vector(n->next_scale);
  a.out = n->out; a.h = n->h; a.ry = n->ry; a.ru = n->ru;
  a.depth = p.depth; a.slot_bytes = p.slot_bytes;
  const int blocks = std::min((n->rows + s.groups - 1) / s.groups, 148 * p.resident);
  return launch_types(a, n->x_dtype, n->y_dtype, s, NormLaunch{false, post, pre, false, blocks, s.threads(), p.smem, stream});
}

extern "C" int vb_block_norm_backward(const VbBlockNorm* n, const VbBlockNormGrads* g, cudaStream_t stream) {
  const bool post = n->y != nullptr, pre = g->dh != nullptr;
  if (n->rows < 0 || n->tokens < 1 || n->rows % n->tokens || (!post && !pre) || (post && n->ry == nullptr) ||
      (pre && (n->ru == nullptr || n->x == nullptr)) || (!pre && g->dout == nullptr) || !vector_ok(n->weight, n->cols) ||
      !vector_ok(n->gate, n->cols) || !vector_ok(n->next_weight, n->cols) || !vector_ok(n->next_scale, n->cols))
    return (int)cudaErrorInvalidValue;
  const bool wide = n->cols % 8 == 0 && on16(n->x) && on16(n->y) && on16(g->dout) && on16(g->dh) && on16(g->dx) && on16(g->dy);
  if (n->rows == 0) return 0;
  const bool dout = g->dout != nullptr;
  NormShape s;
  NormPlan p;
  int blocks;
  if (!backward_plan(n->rows, n->cols, n->tokens, dtype_size(n->x_dtype) * ((pre ? 1 : 0) + (dout ? 1 : 0)),
                     dtype_size(n->y_dtype) * ((post ? 1 : 0) + (pre ? 1 : 0)), wide, s, p, blocks))
    return (int)cudaErrorInvalidValue;
  NormSumArgs t{};
  t.weight[0] = to_vector(n->weight); t.partner[0] = to_vector(n->gate);
  t.weight[1] = to_vector(n->next_weight); t.partner[1] = to_vector(n->next_scale);
  if (post) { t.dweight[0] = g->dweight; t.dpartner[0] = g->dgate; }
  if (pre) { t.dweight[1] = g->dnext_weight; t.dpartner[1] = g->dnext_scale; }
  if (n->tokens == n->rows) t.partner[0].pitch = t.partner[1].pitch = 0;      // one sample: its vectors are shared by all rows
  bool shared = false, per_sample = false;
  for (int k = 0; k < 2; ++k) {
    shared = shared || t.dweight[k] != nullptr || (t.dpartner[k] != nullptr && t.partner[k].pitch == 0);
    per_sample = per_sample || (t.dpartner[k] != nullptr && t.partner[k].pitch != 0);
  }
  if ((shared || per_sample) && (g->workspace == nullptr || !on16(g->workspace) ||
                                 g->workspace_floats < backward_floats(s, blocks, n->rows, n->cols, n->tokens)))
    return (int)cudaErrorInvalidValue;
  NormArgs a{};
  a.rows = n->rows; a.cols = n->cols; a.tokens = n->tokens; a.warps = s.warps;
  a.alpha = n->residual_scale; a.eps = n->eps;
  a.x = n->x; a.y = n->y;
  a.weight = t.weight[0]; a.gate = t.partner[0];
  a.next_weight = t.weight[1]; a.next_scale = t.partner[1];
  a.ry = n->ry; a.ru = n->ru;
  a.dout = g->dout; a.dh = g->dh; a.dx = g->dx; a.dy = g->dy;
  a.sums = shared ? g->workspace : nullptr;
  a.parked = g->workspace + (shared ? (long long)blocks * 2 * n->cols : 0);
  if (t.partner[0].pitch != 0) a.dgate = t.dpartner[0];
  if (t.partner[1].pitch != 0) a.dnext_scale = t.dpartner[1];
  a.depth = p.depth; a.slot_bytes = p.slot_bytes;
  const int rc = launch_types(a, n->x_dtype, n->y_dtype, s,
                              NormLaunch{true, post, pre, n->tokens < n->rows, blocks, s.threads(), p.smem, stream});
  if (rc != 0 || !(shared || per_sample)) return rc;
  t.rows = n->rows; t.cols = n->cols; t.tokens = n->tokens;
  t.blocks = shared ? blocks : 0;
  t.units = std::min((long long)blocks * s.groups, (long long)n->rows);
  t.sums = a.sums; t.parked = a.parked;
  const long long boundaries = per_sample ? (t.units + 2) / 4 : 0;      // units - 1 of them, four to a block
  if (boundaries + t.blocks > 0)
    norm_sums_kernel<<<dim3((unsigned)boundaries + (shared ? 1 : 0), (n->cols + 127) / 128), 1024, 0, stream>>>(t);
  return (int)cudaGetLastError();
}
