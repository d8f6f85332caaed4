// Kernels of block_norm.cu and their launches; one source file per pair of stream and branch types instantiates them.
#pragma once
#include <atomic>
#include <climits>

#include "api.h"
#include "common/launch.cuh"
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
  int totals_shared;           // where sums of several samples meet: 1 in shared memory, 0 in `sums` itself (one group to a block)
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

// A piece: eight neighbouring values of a row as they are stored, one or two 16-byte words.  SHIFT kernels take rows whose
// pieces do not start on 16-byte boundaries (odd widths, offset views) or whose last piece is cut off: they read and write
// the aligned words around a piece and shift the bytes into place.
constexpr int kPiece = 8;
template <typename T> struct Piece {
  static constexpr int kWords = kPiece * (int)sizeof(T) / 16;
  union {
    T value[kPiece];
    uint4 word[kWords];
    uint32_t reg[4 * kWords];
  };
  __device__ __forceinline__ Piece() {}
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) word[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void load_part(const T* p, int count) {        // single values, zeros behind them
    clear();
#pragma unroll
    for (int i = 0; i < kPiece; ++i)
      if (i < count) value[i] = p[i];
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4 * kWords; ++i) reg[i] = 0u;
  }
  __device__ __forceinline__ float get(int i) const { return as_float(value[i]); }
  __device__ __forceinline__ void set(int i, float v) { assign(value[i], v); }
};

template <typename T> __device__ __forceinline__ int misalignment(const T* row) { return (int)(reinterpret_cast<uintptr_t>(row) & 15); }

// words[k] becomes the 32-bit word at byte `offset` + 4 k of `words`, for the first N of them; `offset` is even, at most 16,
// and the same for the whole warp
template <int N, int M> __device__ __forceinline__ void shift_bytes(uint32_t (&words)[M], int offset) {
  static_assert(M >= N + 4, "the words behind the last one are shifted in");
  if (offset & 16) {
#pragma unroll
    for (int k = 0; k < N; ++k) words[k] = words[k + 4];
  }
  if (offset & 8) {
#pragma unroll
    for (int k = 0; k < N + 2; ++k) words[k] = words[k + 2];
  }
  if (offset & 4) {
#pragma unroll
    for (int k = 0; k < N + 1; ++k) words[k] = words[k + 1];
  }
  if (offset & 2) {
#pragma unroll
    for (int k = 0; k < N; ++k) words[k] = __funnelshift_r(words[k], words[k + 1], 16);
  }
}

// Writes the pieces of a warp's neighbouring columns; every lane takes part, those without columns with `active` false.
// SHIFT: a lane writes the aligned words that begin in the piece before its own (whose end it gets from the lane below);
// values of words that are not whole in the warp are written one by one.
template <typename T, bool SHIFT>
__device__ __forceinline__ void store_piece(T* row, int c, int cols, bool active, const Piece<T>& piece) {
  constexpr int kWords = Piece<T>::kWords;
  if constexpr (!SHIFT) {
    if (active) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) reinterpret_cast<uint4*>(row + c)[i] = piece.word[i];
    }
  } else {
    const int lane = threadIdx.x & 31, r = misalignment(row), size = (int)sizeof(T);
    const int begin = c * size - r, end = cols * size;           // of the first word, relative to the row; of the row
    uint32_t words[4 * kWords + 4];
#pragma unroll
    for (int k = 0; k < 4; ++k) words[k] = __shfl_up_sync(kAll, piece.reg[4 * (kWords - 1) + k], 1);
#pragma unroll
    for (int k = 0; k < 4 * kWords; ++k) words[4 + k] = piece.reg[k];
    shift_bytes<4 * kWords>(words, 16 - r);
    bool whole[kWords + 1];
#pragma unroll
    for (int g = 0; g <= kWords; ++g) whole[g] = active && begin + 16 * g + 16 <= end;
    whole[0] = whole[0] && (r == 0 || lane > 0);
    whole[kWords] = whole[kWords] && lane < 31;                  // the next lane's first word
    char* at = reinterpret_cast<char*>(row) + begin;
#pragma unroll
    for (int g = 0; g < kWords; ++g)
      if (whole[g]) *reinterpret_cast<uint4*>(at + 16 * g) = make_uint4(words[4 * g], words[4 * g + 1], words[4 * g + 2], words[4 * g + 3]);
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
      const int g = (i * size + r) >> 4;
      bool covered = whole[0];
#pragma unroll
      for (int k = 1; k <= kWords; ++k) covered = g == k ? whole[k] : covered;
      if (active && c + i < cols && !covered) row[c + i] = piece.value[i];
    }
  }
}

// ---- fetching rows ahead -------------------------------------------------------------------------------------------
// A thread copies the pieces of the next rows that it will need itself into its own 16-byte places in shared memory
// (cp.async), so nothing but its own copies has to be waited for: no barrier, and no registers hold the rows in flight.
__device__ __forceinline__ void copy_ahead(uint32_t to, const void* from, bool through_l1) {
  if (through_l1) asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// the first `bytes` of a word, zeros behind them
__device__ __forceinline__ void copy_ahead_part(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copy_wait(int pending) {     // all but the youngest `pending` groups have arrived
  if (pending >= 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
  else if (pending == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 1;" ::: "memory");
}

// One tensor's part of a slot: V pieces per thread, 16-byte words of neighbouring threads next to each other.  SHIFT: the
// words around a piece, one more than it has; neighbours fetch the word they share both, the second time from L1.
template <typename T, int V, bool SHIFT> struct Strip {
  static constexpr int kWords = Piece<T>::kWords + (SHIFT ? 1 : 0);
  __device__ __forceinline__ static int bytes(int threads) { return V * kWords * threads * 16; }
  // fp32 pieces are two words apart in memory: the halves of a 32-byte sector meet in L1
  __device__ __forceinline__ static void fetch(uint32_t slot, const T* row, int tid, int threads, int cols) {
    const int r = SHIFT ? misalignment(row) : 0;
    const char* base = reinterpret_cast<const char*>(row) - r;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (tid + j * threads) * kPiece;
      if (c < cols) {
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          const uint32_t to = slot + ((j * kWords + w) * threads + tid) * 16;
          const int from = c * (int)sizeof(T) + 16 * w;
          if constexpr (SHIFT) {
            const int left = r + cols * (int)sizeof(T) - from;   // of the row from this word on; nothing behind it is read
            copy_ahead_part(to, base + (left > 0 ? from : 0), max(0, min(left, 16)));
          } else {
            copy_ahead(to, base + from, kWords > 1);
          }
        }
      }
    }
  }
  __device__ __forceinline__ static void take(const unsigned char* slot, int j, int tid, int threads, int r, Piece<T>& piece) {
    uint32_t words[4 * kWords + 4];
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      const uint4 v = *reinterpret_cast<const uint4*>(slot + ((j * kWords + w) * threads + tid) * 16);
      words[4 * w] = v.x; words[4 * w + 1] = v.y; words[4 * w + 2] = v.z; words[4 * w + 3] = v.w;
    }
    if constexpr (SHIFT) shift_bytes<4 * Piece<T>::kWords>(words, r);
#pragma unroll
    for (int k = 0; k < 4 * Piece<T>::kWords; ++k) piece.reg[k] = words[k];
  }
};

// Sums over the warps of a row; every thread gets them.  `turn` alternates between two buffers, so that one barrier per
// call is enough: a warp can only reach the buffer's next use through the other buffer's barrier.  Rows that a block works
// on at the same time meet at barriers of their own (named one by one: a barrier number in a register would reserve all
// sixteen for the block).
__device__ __forceinline__ void row_barrier(int warps, int group) {
  if (group == 0) asm volatile("bar.sync 1, %0;" ::"r"(warps * 32) : "memory");
  else if (group == 1) asm volatile("bar.sync 2, %0;" ::"r"(warps * 32) : "memory");
  else if (group == 2) asm volatile("bar.sync 3, %0;" ::"r"(warps * 32) : "memory");
  else asm volatile("bar.sync 4, %0;" ::"r"(warps * 32) : "memory");
}
__device__ __forceinline__ float row_sum(float v, int warps, int group, float (*buffer)[32], int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  if (warps == 1) return v;
  const int lane = threadIdx.x & 31, first = group * warps;
  if (lane == 0) buffer[turn][threadIdx.x >> 5] = v;
  row_barrier(warps, group);
  if (warps <= 4) {
    v = buffer[turn][first] + buffer[turn][first + 1];
    if (warps > 2) v += buffer[turn][first + 2];
    if (warps > 3) v += buffer[turn][first + 3];
  } else {                                      // at most 16; every warp adds the warps' sums for itself
    v = (lane & 15) < warps ? buffer[turn][first + (lane & 15)] : 0.f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  }
  turn ^= 1;
  return v;
}
// Three sums at once: the first two exchanges leave every eight lanes with one of them, so that three values cost 6 shuffles
// and not 15, and the sums of up to 16 warps 10 (8 warps: 6).
__device__ __forceinline__ void row_sum(float (&v)[3], int warps, int group, float (*buffer)[3][32], int& turn) {
  const int lane = threadIdx.x & 31, first = group * warps;
  const bool upper = lane & 16, odd = lane & 8;
  float x = __shfl_xor_sync(kAll, upper ? v[0] : v[2], 16), y = __shfl_xor_sync(kAll, v[1], 16);
  x += upper ? v[2] : v[0];                     // lanes 0-15: the first sum, 16-31: the third
  y = upper ? 0.f : y + v[1];                   // lanes 0-15: the second
  float keep = (odd ? y : x) + __shfl_xor_sync(kAll, odd ? x : y, 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) keep += __shfl_xor_sync(kAll, keep, o);
  if (warps > 1) {
    if (lane < 24 && (lane & 7) == 0) buffer[turn][lane >> 3][threadIdx.x >> 5] = keep;
    row_barrier(warps, group);
    if (warps <= 8) {
      keep = lane < 24 && (lane & 7) < warps ? buffer[turn][lane >> 3][first + (lane & 7)] : 0.f;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) keep += __shfl_xor_sync(kAll, keep, o);
    } else {
      const bool there = (lane & 15) < warps;
      keep = there ? buffer[turn][lane >> 4][first + (lane & 15)] : 0.f;
      float third = there ? buffer[turn][2][first + (lane & 15)] : 0.f;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) {
        keep += __shfl_xor_sync(kAll, keep, o);
        third += __shfl_xor_sync(kAll, third, o);
      }
      v[0] = __shfl_sync(kAll, keep, 0);
      v[1] = __shfl_sync(kAll, keep, 16);
      v[2] = third;
      turn ^= 1;
      return;
    }
    turn ^= 1;
  }
  v[0] = __shfl_sync(kAll, keep, 0);
  v[1] = __shfl_sync(kAll, keep, 8);
  v[2] = __shfl_sync(kAll, keep, 16);
}

// fp32 values of a thread's columns in shared memory, in places of its own (no barrier): value i of piece j
__device__ __forceinline__ int own_place(int j, int i, int tid, int threads) {
  return ((j * (kPiece / 4) + i / 4) * threads + tid) * 4 + i % 4;
}
__device__ __forceinline__ void own_values(const float* area, int j, int tid, int threads, float (&v)[kPiece]) {
#pragma unroll
  for (int w = 0; w < kPiece / 4; ++w) {
    const float4 f = *reinterpret_cast<const float4*>(area + own_place(j, 4 * w, tid, threads));
    v[4 * w] = f.x; v[4 * w + 1] = f.y; v[4 * w + 2] = f.z; v[4 * w + 3] = f.w;
  }
}

__device__ __forceinline__ float vector_value(const NormVector& v, long long sample, int c, float shift, float otherwise) {
  return v.data != nullptr ? shift + load_as_float(v.data, sample * v.pitch + c, v.dtype) : otherwise;
}
// the values of a piece's columns of an optional vector (absent: 1) plus `shift`; behind the last column 0
__device__ __forceinline__ void vector_values(const NormVector& v, long long sample, int c, int cols, float shift, float (&f)[kPiece]) {
  if (v.data == nullptr) {
#pragma unroll
    for (int i = 0; i < kPiece; ++i) f[i] = 1.f;
    return;
  }
  const long long at = sample * v.pitch + c;
  if (v.wide && c + kPiece <= cols) {
    if (v.dtype == kF32) {
      Piece<float> raw;
      raw.load(reinterpret_cast<const float*>(v.data) + at);
#pragma unroll
      for (int i = 0; i < kPiece; ++i) f[i] = raw.get(i) + shift;
    } else {
      Piece<__nv_bfloat16> raw;
      raw.load(reinterpret_cast<const __nv_bfloat16*>(v.data) + at);
#pragma unroll
      for (int i = 0; i < kPiece; ++i)
        f[i] = (v.dtype == kBF16 ? raw.get(i) : __half2float(__ushort_as_half(__bfloat16_as_ushort(raw.value[i])))) + shift;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPiece; ++i) f[i] = c + i < cols ? load_as_float(v.data, at + i, v.dtype) + shift : 0.f;
  }
}

// product of two optional vectors (the second plus `shift`) for the columns of one thread; once per sample
template <int V>
__device__ __forceinline__ void store_gain(const NormVector& a, const NormVector& b, float shift, long long sample, int tid,
                                           int threads, int cols, float* area) {
#pragma unroll 1
  for (int j = 0; j < V; ++j) {
    const int c = (tid + j * threads) * kPiece;
    if (c < cols) {
      float f[kPiece], g[kPiece];
      vector_values(a, sample, c, cols, 0.f, f);
      vector_values(b, sample, c, cols, shift, g);
#pragma unroll
      for (int i = 0; i < kPiece; ++i) area[own_place(j, i, tid, threads)] = f[i] * g[i];
    }
  }
}

// A row's values stay in registers through both norms: one read, one write.  Bound by memory: 4 x 8192 x 4096 bf16 202 us
// (81 % of the copy rate), 128 x 256 x 1152 with an fp32 stream 88 us (78 %).
template <typename TX, typename TY, bool SHIFT, int V, int THREADS, bool POST, bool PRE>
__global__ void __launch_bounds__(THREADS)
norm_forward_kernel(const NormArgs a) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float buffer[2][32];
  using SX = Strip<TX, V, SHIFT>;
  using SY = Strip<TY, V, SHIFT>;
  const int threads = a.warps * 32, group = threadIdx.x / threads, tid = threadIdx.x - group * threads;
  const int groups = blockDim.x / threads, units = gridDim.x * groups;
  const int per_unit = (int)(((unsigned)a.rows + units - 1u) / units);        // up to 2^31 - 1 rows
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
  float* gains = reinterpret_cast<float*>(ring + (size_t)groups * slots * a.slot_bytes) + (size_t)group * 2 * V * kPiece * threads;
  float* next_gains = gains + V * kPiece * threads;
  long long sample = first / a.tokens, sample_end = first;
  int turn = 0, head = 0;
  for (long long row = first; row < last; ++row) {
    Piece<TX> px[V];
    Piece<TY> py[V];
    const long long base = row * a.cols;
    if (a.depth > 0) {
      const int ahead = head + a.depth;
      fetch(row + a.depth, ahead >= slots ? ahead - slots : ahead);
      copy_wait(a.depth);
      const unsigned char* slot = mine + head * a.slot_bytes;
      head = head + 1 == slots ? 0 : head + 1;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        SX::take(slot, j, tid, threads, misalignment(x + base), px[j]);
        if (POST) SY::take(slot + x_bytes, j, tid, threads, misalignment(y + base), py[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = (tid + j * threads) * kPiece;
        if (c < a.cols) {
          if constexpr (SHIFT) {
            px[j].load_part(x + base + c, a.cols - c);
            if (POST) py[j].load_part(y + base + c, a.cols - c);
          } else {
            px[j].load(x + base + c);
            if (POST) py[j].load(y + base + c);
          }
        }
      }
    }
    if (row >= sample_end) {
      if (row > first) ++sample;
      sample_end = (sample + 1) * a.tokens;
      if (POST) store_gain<V>(a.weight, a.gate, 0.f, sample, tid, threads, a.cols, gains);
      if (PRE) store_gain<V>(a.next_weight, a.next_scale, 1.f, sample, tid, threads, a.cols, next_gains);
    }
    float u[V][kPiece], sum = 0.f;
    if (POST) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if ((tid + j * threads) * kPiece < a.cols)
#pragma unroll
          for (int i = 0; i < kPiece; ++i) sum = fmaf(py[j].get(i), py[j].get(i), sum);
      const float ry = rsqrtf(fmaf(row_sum(sum, a.warps, group, buffer, turn), inverse, a.eps));
      if (tid == 0 && a.ry != nullptr) a.ry[row] = ry;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = (tid + j * threads) * kPiece;
        Piece<TX> o;
        if (c < a.cols) {
          float gain[kPiece];
          own_values(gains, j, tid, threads, gain);
#pragma unroll
          for (int i = 0; i < kPiece; ++i) {
            u[j][i] = fmaf(a.alpha, px[j].get(i), py[j].get(i) * ry * gain[i]);
            o.set(i, u[j][i]);
          }
        }
        store_piece<TX, SHIFT>(reinterpret_cast<TX*>(a.out) + base, c, a.cols, c < a.cols, o);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < kPiece; ++i) u[j][i] = px[j].get(i);
    }
    if (PRE) {
      sum = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if ((tid + j * threads) * kPiece < a.cols)
#pragma unroll
          for (int i = 0; i < kPiece; ++i) sum = fmaf(u[j][i], u[j][i], sum);
      const float ru = rsqrtf(fmaf(row_sum(sum, a.warps, group, buffer, turn), inverse, a.eps));
      if (tid == 0 && a.ru != nullptr) a.ru[row] = ru;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = (tid + j * threads) * kPiece;
        Piece<TY> o;
        if (c < a.cols) {
          float gain[kPiece];
          own_values(next_gains, j, tid, threads, gain);
#pragma unroll
          for (int i = 0; i < kPiece; ++i) o.set(i, u[j][i] * ru * gain[i]);
        }
        store_piece<TY, SHIFT>(reinterpret_cast<TY*>(a.h) + base, c, a.cols, c < a.cols, o);
      }
    }
  }
}

// Bound by the latency of a row's load, reduction and store one after the other where few rows are in flight, by issued
// instructions elsewhere: 4 x 8192 x 4096 bf16 349 us (70 % of the copy rate), 128 x 256 x 1152 with an fp32 stream 146 us
// (71 %).  Wider rows spill, as d, yh, uh and the two column sums wait for the row's sums in registers: two pieces a thread (more
// than 4096 columns) 80 to 128 bytes, four (more than 8192) 464 to 736, shifted 96 to 272 and 1320 to 1832.  2 x 4096 x 8192 bf16
// takes 181 us (68 %), 2 x 2048 x 16384 351 (35 %).
// With q = gate * weight * yh, t = dh * next_weight * (1 + next_scale), uh = u * ru, c = mean(t uh):
//   d  = dout + ru (t - uh c)                  the gradient of u
//   dx = alpha d,   dy = ry (d gate weight - yh m),   m = mean(d q)
// mean(d q) = mean((dout + ru t) q) - ru c mean(uh q), so one reduction of three sums per row serves both norms.
//
// Column sums S = sum of d * yh and R = sum of dh * uh give the gradients of the vectors.  Every row group (a block, or
// part of one where rows are short) takes an equal share of consecutive rows.  With several samples, at the end of one it writes
// the gradients of the per-sample vectors if it had the whole sample, else parks the sums (place 0: the sample began in
// an earlier group, 1: it goes on in a later one), and adds them, weighted with the per-sample partner, to the sums of
// the shared vectors.
template <typename TX, typename TY, bool SHIFT, int V, int THREADS, bool POST, bool PRE>
__global__ void __launch_bounds__(THREADS)
norm_backward_kernel(const NormArgs a) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float buffer[2][3][32];
  using SX = Strip<TX, V, SHIFT>;
  using SY = Strip<TY, V, SHIFT>;
  cudaTriggerProgrammaticLaunchCompletion();    // the kernel of the vectors' sums may start when there is room; it waits for this one
  const int threads = a.warps * 32, group = threadIdx.x / threads, tid = threadIdx.x - group * threads;
  const int groups = blockDim.x / threads;
  const TX* x = reinterpret_cast<const TX*>(a.x);
  const TY* y = reinterpret_cast<const TY*>(a.y);
  const TX* dout = reinterpret_cast<const TX*>(a.dout);
  const TY* dh = reinterpret_cast<const TY*>(a.dh);
  const float inverse = 1.f / (float)a.cols;
  const bool samples = a.tokens < a.rows;
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

  float post_sum[V][kPiece], pre_sum[V][kPiece];
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int i = 0; i < kPiece; ++i) post_sum[j][i] = pre_sum[j][i] = 0.f;
  // per group: gains, next gains; then, where sums of several samples or groups meet, sums of S and R
  const int area = V * kPiece * threads;
  float* gains = reinterpret_cast<float*>(ring + (size_t)groups * slots * a.slot_bytes) + (size_t)group * 2 * area;
  float* next_gains = gains + area;
  float* total = reinterpret_cast<float*>(ring + (size_t)groups * slots * a.slot_bytes) + (size_t)(groups + group) * 2 * area;
  if (samples && a.totals_shared) {              // places that the thread itself adds to: no barrier
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < kPiece; ++i) total[own_place(j, i, tid, threads)] = total[area + own_place(j, i, tid, threads)] = 0.f;
  }
  const long long first_sample = samples ? first / a.tokens : 0;
  auto finish_norm = [&](int n, long long sample, const NormVector& weight, const NormVector& partner, float shift, void* grad,
                         float (&sum)[V][kPiece]) {
    const bool fresh = sample == first_sample, before = sample * a.tokens < first, after = (sample + 1) * a.tokens > last;
    float* park = a.parked + ((unit * 2 + (before ? 0 : 1)) * 2 + n) * a.cols;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (tid + j * threads) * kPiece;
      if (c < a.cols) {
        float f[kPiece];
        if (grad != nullptr) {
          if (before || after) {
#pragma unroll
            for (int i = 0; i < kPiece; ++i)
              if (!SHIFT || c + i < a.cols) park[c + i] = sum[j][i];
          } else {
            vector_values(weight, 0, c, a.cols, 0.f, f);
#pragma unroll
            for (int i = 0; i < kPiece; ++i)
              if (!SHIFT || c + i < a.cols) store_from_float(grad, sample * a.cols + c + i, partner.dtype, sum[j][i] * f[i]);
          }
        }
        if (a.sums != nullptr) {
          if (partner.pitch != 0) {
            vector_values(partner, sample, c, a.cols, shift, f);
          } else {
#pragma unroll
            for (int i = 0; i < kPiece; ++i) f[i] = 1.f;
          }
          if (a.totals_shared) {
#pragma unroll
            for (int i = 0; i < kPiece; ++i) total[n * area + own_place(j, i, tid, threads)] += sum[j][i] * f[i];
          } else {
            float* to = a.sums + ((long long)blockIdx.x * 2 + n) * a.cols + c;
#pragma unroll
            for (int i = 0; i < kPiece; ++i)
              if (!SHIFT || c + i < a.cols) to[i] = (fresh ? 0.f : to[i]) + sum[j][i] * f[i];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kPiece; ++i) sum[j][i] = 0.f;
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
      if (samples && row > first) finish_sample(sample++);
      sample_end = samples ? (sample + 1) * a.tokens : last;
      if (POST) store_gain<V>(a.weight, a.gate, 0.f, sample, tid, threads, a.cols, gains);
      if (PRE) store_gain<V>(a.next_weight, a.next_scale, 1.f, sample, tid, threads, a.cols, next_gains);
    }
    const unsigned char* slot = mine + head * a.slot_bytes;
    if (a.depth > 0) {
      const int ahead = head + a.depth;
      fetch(row + a.depth, ahead >= slots ? ahead - slots : ahead);
      copy_wait(a.depth);
      head = head + 1 == slots ? 0 : head + 1;
    }
    float d[V][kPiece], yh[V][kPiece], uh[V][kPiece], sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (tid + j * threads) * kPiece;
      Piece<TX> px, pd;
      Piece<TY> py, ph;
      float gain[kPiece], next_gain[kPiece];
      if (c < a.cols) {
        if (POST) own_values(gains, j, tid, threads, gain);
        if (PRE) own_values(next_gains, j, tid, threads, next_gain);
        if (a.dout == nullptr) pd.clear();
        if (a.depth > 0) {
          if (PRE) SX::take(slot, j, tid, threads, misalignment(x + base), px);
          if (a.dout != nullptr) SX::take(slot + at_dout, j, tid, threads, misalignment(dout + base), pd);
          if (POST) SY::take(slot + at_y, j, tid, threads, misalignment(y + base), py);
          if (PRE) SY::take(slot + at_dh, j, tid, threads, misalignment(dh + base), ph);
        } else if constexpr (SHIFT) {
          if (PRE) px.load_part(x + base + c, a.cols - c);
          if (POST) py.load_part(y + base + c, a.cols - c);
          if (a.dout != nullptr) pd.load_part(dout + base + c, a.cols - c);
          if (PRE) ph.load_part(dh + base + c, a.cols - c);
        } else {
          if (PRE) px.load(x + base + c);
          if (POST) py.load(y + base + c);
          if (a.dout != nullptr) pd.load(dout + base + c);
          if (PRE) ph.load(dh + base + c);
        }
#pragma unroll
        for (int i = 0; i < kPiece; ++i) {
          float q = 0.f, u;
          d[j][i] = pd.get(i);
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
    row_sum(sum, a.warps, group, buffer, turn);
    const float pull = ru * sum[0] * inverse;                       // ru c
    const float m = POST ? (PRE ? fmaf(-pull, sum[2], sum[1]) : sum[1]) * inverse : 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (tid + j * threads) * kPiece;
      Piece<TX> ox;
      Piece<TY> oy;
      if (c < a.cols) {
        float gain[kPiece];
        if (POST) own_values(gains, j, tid, threads, gain);
#pragma unroll
        for (int i = 0; i < kPiece; ++i) {
          const float whole = PRE ? fmaf(-pull, uh[j][i], d[j][i]) : d[j][i];
          ox.set(i, POST ? a.alpha * whole : whole);
          if (POST) {
            oy.set(i, ry * fmaf(-m, yh[j][i], whole * gain[i]));
            post_sum[j][i] = fmaf(whole, yh[j][i], post_sum[j][i]);
          }
        }
        if constexpr (!SHIFT) {
          if (a.dx != nullptr) store_piece<TX, SHIFT>(reinterpret_cast<TX*>(a.dx) + base, c, a.cols, true, ox);
          if (POST && a.dy != nullptr) store_piece<TY, SHIFT>(reinterpret_cast<TY*>(a.dy) + base, c, a.cols, true, oy);
        }
      }
      if constexpr (SHIFT) {
        if (a.dx != nullptr) store_piece<TX, SHIFT>(reinterpret_cast<TX*>(a.dx) + base, c, a.cols, c < a.cols, ox);
        if (POST && a.dy != nullptr) store_piece<TY, SHIFT>(reinterpret_cast<TY*>(a.dy) + base, c, a.cols, c < a.cols, oy);
      }
    }
  }
  if (samples && first < last) finish_sample(sample);
  if (a.sums == nullptr || (samples && !a.totals_shared)) return;
  float* to = a.sums + (long long)blockIdx.x * 2 * a.cols;
  if (!samples && groups == 1) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (tid + j * threads) * kPiece;
      if (c < a.cols)
#pragma unroll
        for (int i = 0; i < kPiece; ++i) {
          if (SHIFT && c + i >= a.cols) continue;
          to[c + i] = POST ? post_sum[j][i] : 0.f;
          to[a.cols + c + i] = PRE ? pre_sum[j][i] : 0.f;
        }
    }
    return;
  }
  if (!samples) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        total[own_place(j, i, tid, threads)] = POST ? post_sum[j][i] : 0.f;
        total[area + own_place(j, i, tid, threads)] = PRE ? pre_sum[j][i] : 0.f;
      }
  }
  __syncthreads();
  // the first group adds the groups' sums in order
  if (group == 0) {
#pragma unroll 1
    for (int k = 0; k < 2 * V * kPiece; ++k) {
      const int n = k / (V * kPiece), j = k / kPiece % V, i = k % kPiece, c = (tid + j * threads) * kPiece + i;
      if (c < a.cols) {
        const float* from = total + n * area + own_place(j, i, tid, threads);
        float s = from[0];
        for (int g = 1; g < groups; ++g) s += from[(size_t)g * 2 * area];
        to[n * a.cols + c] = s;
      }
    }
  }
}

constexpr int kSharedPerBlock = 227 * 1024;

struct NormShape {
  bool shift;                  // pieces do not all start on 16-byte boundaries, or the last is cut off
  int v, warps, groups;        // pieces per thread, warps per row, rows a block works on at a time
  int bound;                   // threads that the kernel's template is built for
  int threads() const { return warps * groups * 32; }
};

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
  bool backward, post, pre;
  int blocks, threads;         // blocks: as many as there is room for, at most these
  size_t smem;
  cudaStream_t stream;
};

// blocks of a kernel that one SM holds at once; the answer for the last shape is kept
template <auto Kernel>
int resident_blocks(int threads, size_t smem) {
  static std::atomic<unsigned long long> last{0};      // threads (16 bits), smem (32), blocks (16)
  const unsigned long long key = (unsigned long long)threads << 48 | (unsigned long long)smem << 16;
  const unsigned long long seen = last.load(std::memory_order_relaxed);
  if ((seen & ~0xffffull) == key) return (int)(seen & 0xffffull);
  int blocks = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, Kernel, threads, smem) != cudaSuccess) return 1;
  blocks = blocks > 1 ? blocks : 1;
  last.store(key | (unsigned long long)blocks, std::memory_order_relaxed);
  return blocks;
}

// one wave; returns the number of blocks
template <auto Kernel>
int launch_kernel(const NormArgs& a, const NormLaunch& l) {
  if (l.smem > 48 * 1024 - 1024) allow_shared<Kernel>();
  const int room = 148 * resident_blocks<Kernel>(l.threads, l.smem), blocks = l.blocks < room ? l.blocks : room;
  Kernel<<<blocks, l.threads, l.smem, l.stream>>>(a);
  count_launch();
  return blocks;
}

template <bool BACKWARD, typename TX, typename TY, bool SHIFT, int V, int THREADS>
int launch_norms(const NormArgs& a, const NormLaunch& l) {
  if constexpr (BACKWARD) {
    if (l.post && l.pre) return launch_kernel<norm_backward_kernel<TX, TY, SHIFT, V, THREADS, true, true>>(a, l);
    if (l.post) return launch_kernel<norm_backward_kernel<TX, TY, SHIFT, V, THREADS, true, false>>(a, l);
    return launch_kernel<norm_backward_kernel<TX, TY, SHIFT, V, THREADS, false, true>>(a, l);
  } else {
    if (l.post && l.pre) return launch_kernel<norm_forward_kernel<TX, TY, SHIFT, V, THREADS, true, true>>(a, l);
    if (l.post) return launch_kernel<norm_forward_kernel<TX, TY, SHIFT, V, THREADS, true, false>>(a, l);
    return launch_kernel<norm_forward_kernel<TX, TY, SHIFT, V, THREADS, false, true>>(a, l);
  }
}

template <typename TX, typename TY, bool SHIFT>
int launch_aligned(const NormArgs& a, const NormShape& s, const NormLaunch& l) {
  if (l.backward) {
    if (s.v == 1) return launch_norms<true, TX, TY, SHIFT, 1, 512>(a, l);
    if (s.v == 2) return launch_norms<true, TX, TY, SHIFT, 2, 512>(a, l);
    return launch_norms<true, TX, TY, SHIFT, 4, 512>(a, l);
  } else {
    if (s.v == 1) return launch_norms<false, TX, TY, SHIFT, 1, 256>(a, l);
    if (s.v == 2) return launch_norms<false, TX, TY, SHIFT, 2, 256>(a, l);
    if (s.v == 3) return launch_norms<false, TX, TY, SHIFT, 3, 256>(a, l);
    if (s.bound == 256) return launch_norms<false, TX, TY, SHIFT, 4, 256>(a, l);
    return launch_norms<false, TX, TY, SHIFT, 4, 512>(a, l);
  }
}

template <typename TX, typename TY>
int launch_shape(const NormArgs& a, const NormShape& s, const NormLaunch& l) {
  return s.shift ? launch_aligned<TX, TY, true>(a, s, l) : launch_aligned<TX, TY, false>(a, s, l);
}

}  // namespace vb
