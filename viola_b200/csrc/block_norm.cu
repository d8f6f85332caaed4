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

#include "block_norm.cuh"
#include "common/launch.cuh"

namespace vb {

extern template int launch_shape<float, float>(const NormArgs&, const NormShape&, const NormLaunch&);
extern template int launch_shape<float, __nv_bfloat16>(const NormArgs&, const NormShape&, const NormLaunch&);
extern template int launch_shape<float, __half>(const NormArgs&, const NormShape&, const NormLaunch&);
extern template int launch_shape<__nv_bfloat16, __nv_bfloat16>(const NormArgs&, const NormShape&, const NormLaunch&);
extern template int launch_shape<__half, __half>(const NormArgs&, const NormShape&, const NormLaunch&);

struct NormSumArgs {
  int rows, cols, tokens;
  int blocks;                  // sets of sums, 0 if nothing is shared
  long long units;             // row groups of the backward kernel that have rows
  int by_sample;               // places are samples, else group boundaries
  const float *sums, *parked;
  NormVector weight[2], partner[2];          // of the two norms: weight, and gate / next_scale
  void *dweight[2], *dpartner[2];            // gradients, or null
};

// Gradients of the vectors from what the row groups left.  The shared ones: with T the sum of the blocks' sums, T for a
// weight whose partner is per sample (its factors are in T), partner * T for one whose partner is shared, and weight * T
// for a shared partner.  Per-sample ones of samples that several groups shared: weight * sum of what they parked.
// A block has one norm and 128 columns, 4 a thread, and 16 rows of threads: the first block of a column range (where anything
// is shared) gives all of them to T, every other one eight to each of two samples, or of two group boundaries where there are
// fewer of those; the first boundary inside a sample takes that sample.  A row takes every 16th (8th) set, and the rows are
// added in order.  What bounds it is the latency of the loads for T, one set of every block of the backward kernel (444 for
// 128 x 256 x 1152), so a thread has eight under way:
// the sums of 7175 x 1001 fp16 in 592 groups take 6 us less than with one after the other (46 to 40 us of the pass).
constexpr int kAhead = 8;
__global__ void __launch_bounds__(512)
norm_sums_kernel(const NormSumArgs a) {
  __shared__ float4 part[16][32];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, c = blockIdx.y * 128 + lane * 4, n = blockIdx.z;
  const int has_shared = a.blocks > 0 ? 1 : 0;
  const bool shared_block = has_shared && blockIdx.x == 0;
  const int stride = shared_block ? 16 : 8, turn = shared_block ? row : row % 8;
  const bool per_sample = a.partner[n].pitch != 0;
  if (!(shared_block ? a.dweight[n] != nullptr || (a.dpartner[n] != nullptr && !per_sample)
                     : a.dpartner[n] != nullptr && per_sample))
    return;                                     // the whole block
  const float* from = a.sums;
  long long sample = 0, first = 0, last = a.blocks;
  if (!shared_block) {
    from = a.parked;
    first = last = 0;
    const long long place = ((long long)blockIdx.x - has_shared) * 2 + row / 8;
    // the group that has a row is the last one that begins at or before it
    auto group_of = [&](long long r) -> long long {
      const unsigned long long before = (unsigned long long)(r + 1) * a.units - 1;
      return before >> 32 ? before / a.rows : (unsigned)before / (unsigned)a.rows;
    };
    long long begin = -1;                       // first group of the sample, if others have rows of it too
    if (a.by_sample) {
      sample = place;
      if (sample * a.tokens < a.rows) begin = group_of(sample * a.tokens);
    } else if (place + 1 < a.units) {
      const long long boundary = a.rows * (place + 1) / a.units;
      sample = boundary / a.tokens;
      if (boundary > sample * a.tokens && a.rows * place / a.units <= sample * a.tokens) begin = place;
    }
    if (begin >= 0) {
      const long long end = group_of((sample + 1) * a.tokens - 1);
      if (end > begin) {
        first = begin;
        last = end + 1;
      }
    }
  }
  const NormVector &w = a.weight[n], &p = a.partner[n];
  float by_weight[4] = {}, by_partner[4] = {};  // factors of the sums, read while the sums are on their way
  if (turn == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (c + i >= a.cols) continue;
      by_weight[i] = vector_value(w, 0, c + i, 0.f, 1.f);
      by_partner[i] = per_sample ? 1.f : vector_value(p, 0, c + i, n ? 1.f : 0.f, 1.f);
    }
  }
  cudaGridDependencySynchronize();              // from here on: what the backward kernel wrote
  float total[4] = {0.f, 0.f, 0.f, 0.f};
  const bool wide = a.cols % 4 == 0;
  for (long long u = first + turn; u < last; u += kAhead * stride) {
    float t[kAhead][4];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const long long at = u + k * stride, set = shared_block ? at : at * 2 + (at > first ? 0 : 1);
      const float* sums = from + (set * 2 + n) * a.cols + c;
      const bool there = at < last && c < a.cols;
      if (wide) {
        const float4 v = there ? *reinterpret_cast<const float4*>(sums) : make_float4(0.f, 0.f, 0.f, 0.f);
        t[k][0] = v.x; t[k][1] = v.y; t[k][2] = v.z; t[k][3] = v.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) t[k][i] = there && c + i < a.cols ? sums[i] : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) total[i] += t[k][i];
  }
  part[row][lane] = make_float4(total[0], total[1], total[2], total[3]);
  __syncthreads();
  // the first row of a set (two sets of eight, or one) finishes it
  if (turn > 0 || first >= last) return;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = row; i < row + stride; ++i) {
    const float4 t = part[i][lane];
    sum[0] += t.x; sum[1] += t.y; sum[2] += t.z; sum[3] += t.w;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (c + i >= a.cols) continue;
    if (!shared_block) {
      store_from_float(a.dpartner[n], sample * a.cols + c + i, p.dtype, sum[i] * by_weight[i]);
    } else {
      if (a.dweight[n] != nullptr) store_from_float(a.dweight[n], c + i, w.dtype, sum[i] * by_partner[i]);
      if (a.dpartner[n] != nullptr && !per_sample) store_from_float(a.dpartner[n], c + i, p.dtype, sum[i] * by_weight[i]);
    }
  }
}

}  // namespace vb

using namespace vb;

namespace {

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Forward: the work of a row that does not grow with its values (addresses, reductions) is about that of ten values for
// every thread, so few threads with many values each take the fewest instructions: as many as four pieces a thread, as long
// as not more lanes idle for it (128 x 256 x 1152, fp32 stream: 120 us with one piece a thread, 86 with three; 4 x 8192 x 4096
// bf16: 254 and 202).  Backward: a piece takes three times the registers, and warps to hide latency count for more
// (the same: 154 us with one piece, 171 with two, 237 with three; 356 with one, 380 with two, 530 with four;
// each with 8 us more for the vectors' sums
// than now).  One norm at 80 registers, which makes six warps of a scheduler's four, won at 4 x 8192 x 2048 bf16 (149 to
// 135 us; the norm behind a block takes 144 now, 57 % of the copy rate, the one in front of it 113, 55 %) and lost where more row
// groups leave more sums (7175 x 1001 fp16 47 to 55, 128 x 256 x 1152 101 to 106): not kept.
// Shifted pieces take more registers too: two a thread forward (4 x 4096 x 2047 bf16: 118 us with one, 103 with two, 133
// with four; 100 now).
bool norm_shape(int cols, bool shift, bool backward, NormShape& s) {
  if (cols < 1 || cols > VB_NORM_MAX_COLS || (!shift && cols % kPiece)) return false;
  const int pieces = (cols + kPiece - 1) / kPiece;
  s.shift = shift;
  if (backward) {
    s.v = pieces <= 512 ? 1 : pieces <= 1024 ? 2 : 4;
  } else {
    int best = INT_MAX;
    for (int v = shift && pieces <= 512 ? 2 : 4; v >= 1; --v) {
      const int warps = (pieces + 32 * v - 1) / (32 * v), cost = warps * (kPiece * v + 10);
      if (warps <= (v == 4 ? 16 : 8) && cost < best) {
        best = cost;
        s.v = v;
      }
    }
  }
  s.warps = (pieces + 32 * s.v - 1) / (32 * s.v);
  s.groups = std::max(1, (backward ? 8 : 4) / s.warps);
  s.bound = backward || s.warps > 8 ? 512 : 256;
  return true;
}
// threads that an SM's registers do for
int forward_threads(const NormShape& s) {
  return s.v == 1 ? 768 : s.v == 2 ? 512 : s.v == 3 ? 384 : s.warps > 8 ? 512 : 320;
}
constexpr int kBackwardThreads = 512;

// Rows fetched ahead (as many up to three as cost no resident block), shared memory for them and for `areas` fp32 values
// per column, and blocks that one SM holds where its registers do for `resident_threads`.
struct NormPlan {
  int depth, slot_bytes, resident;
  size_t smem;
};
// blocks that give every row a group
int row_blocks(int rows, const NormShape& s) { return (int)(((long long)rows + s.groups - 1) / s.groups); }
int by_registers(const NormShape& s, int resident_threads) { return std::max(1, resident_threads / s.threads()); }
NormPlan norm_plan(const NormShape& s, int piece_bytes, int areas, int resident_threads) {
  NormPlan p{0, 0, 1, 0};
  const size_t extra = (size_t)areas * s.v * kPiece * s.threads() * sizeof(float);
  const int most = by_registers(s, resident_threads);
  const int slot = s.v * s.warps * 32 * piece_bytes;
  for (p.depth = 3;; --p.depth) {
    p.smem = extra + (p.depth ? (size_t)(p.depth + 1) * s.groups * slot : 0);
    p.resident = std::min(most, (int)(kSharedPerBlock / (p.smem + 2048)));
    if (p.resident == most || p.depth == 0 || (p.depth == 1 && p.resident > 0)) break;
  }
  p.slot_bytes = p.depth ? slot : 0;
  return p;
}

// returns the number of blocks launched, 0 for types that do not go together
int launch_types(const NormArgs& a, int x_dtype, int y_dtype, const NormShape& s, const NormLaunch& l) {
  if (x_dtype == kF32 && y_dtype == kF32) return launch_shape<float, float>(a, s, l);
  if (x_dtype == kF32 && y_dtype == kBF16) return launch_shape<float, __nv_bfloat16>(a, s, l);
  if (x_dtype == kF32 && y_dtype == kF16) return launch_shape<float, __half>(a, s, l);
  if (x_dtype == kBF16 && y_dtype == kBF16) return launch_shape<__nv_bfloat16, __nv_bfloat16>(a, s, l);
  if (x_dtype == kF16 && y_dtype == kF16) return launch_shape<__half, __half>(a, s, l);
  return 0;
}

bool vector_ok(const VbNormVector& v, int cols) {
  return v.data == nullptr || (v.dtype >= kF32 && v.dtype <= kF16 && (v.pitch == 0 || v.pitch >= cols));
}
int dtype_size(int dtype) { return dtype == kF32 ? 4 : 2; }
int piece_bytes(int dtype, bool shift) { return kPiece * dtype_size(dtype) + (shift ? 16 : 0); }      // in a slot
NormVector to_vector(const VbNormVector& v) {
  return NormVector{v.data, v.dtype, on16(v.data) && v.pitch * dtype_size(v.dtype) % 16 == 0, v.pitch};
}

// Shared memory of the backward pass and the most blocks: one wave, at least one row to a group
// Sums of several samples meet in shared memory where row groups share a block or it has the room.
bool totals_in_shared(const NormShape& s, int rows, int tokens) {
  return s.groups > 1 || (tokens < rows && 4 * s.v * kPiece * s.threads() * sizeof(float) <= 64 * 1024);
}
bool backward_plan(int rows, int cols, int tokens, int bytes, bool shift, NormShape& s, NormPlan& p, int& blocks) {
  if (!norm_shape(cols, shift, true, s)) return false;
  p = norm_plan(s, bytes, totals_in_shared(s, rows, tokens) ? 4 : 2, kBackwardThreads);
  blocks = std::min(row_blocks(rows, s), 148 * p.resident);
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
  NormShape s;
  if (!norm_shape(cols, true, true, s)) return 0;
  const int blocks = std::min(row_blocks(rows, s), 148 * by_registers(s, kBackwardThreads));
  return backward_floats(s, blocks, rows, cols, tokens);
}

extern "C" int vb_block_norm(const VbBlockNorm* n, cudaStream_t stream) {
  const bool post = n->y != nullptr, pre = n->h != nullptr;
  if (n->rows < 0 || n->tokens < 1 || n->rows % n->tokens || n->x == nullptr || (!post && !pre) || (post && n->out == nullptr) ||
      !vector_ok(n->weight, n->cols) || !vector_ok(n->gate, n->cols) || !vector_ok(n->next_weight, n->cols) ||
      !vector_ok(n->next_scale, n->cols))
    return (int)cudaErrorInvalidValue;
  NormShape s;
  const bool shift = n->cols % kPiece || !on16(n->x) || !on16(n->y) || !on16(n->out) || !on16(n->h);
  if (!norm_shape(n->cols, shift, false, s)) return (int)cudaErrorInvalidValue;
  if (n->rows == 0) return 0;
  const NormPlan p = norm_plan(s, piece_bytes(n->x_dtype, shift) + (post ? piece_bytes(n->y_dtype, shift) : 0), 2, forward_threads(s));
  NormArgs a{};
  a.rows = n->rows; a.cols = n->cols; a.tokens = n->tokens; a.warps = s.warps;
  a.alpha = n->residual_scale; a.eps = n->eps;
  a.x = n->x; a.y = n->y;
  a.weight = to_vector(n->weight); a.gate = to_vector(n->gate);
  a.next_weight = to_vector(n->next_weight); a.next_scale = to_vector(n->next_scale);
  a.out = n->out; a.h = n->h; a.ry = n->ry; a.ru = n->ru;
  a.depth = p.depth; a.slot_bytes = p.slot_bytes;
  const int blocks = row_blocks(n->rows, s);
  if (launch_types(a, n->x_dtype, n->y_dtype, s, NormLaunch{false, post, pre, blocks, s.threads(), p.smem, stream}) == 0)
    return (int)cudaErrorInvalidValue;
  return (int)cudaGetLastError();
}

extern "C" int vb_block_norm_backward(const VbBlockNorm* n, const VbBlockNormGrads* g, cudaStream_t stream) {
  const bool post = n->y != nullptr, pre = g->dh != nullptr;
  if (n->rows < 0 || n->tokens < 1 || n->rows % n->tokens || (!post && !pre) || (post && n->ry == nullptr) ||
      (pre && (n->ru == nullptr || n->x == nullptr)) || (!pre && g->dout == nullptr) || !vector_ok(n->weight, n->cols) ||
      !vector_ok(n->gate, n->cols) || !vector_ok(n->next_weight, n->cols) || !vector_ok(n->next_scale, n->cols))
    return (int)cudaErrorInvalidValue;
  const bool shift = n->cols % kPiece || !on16(n->x) || !on16(n->y) || !on16(g->dout) || !on16(g->dh) || !on16(g->dx) || !on16(g->dy);
  if (n->rows == 0) return 0;
  const bool dout = g->dout != nullptr;
  NormShape s;
  NormPlan p;
  int blocks;
  const int bytes = piece_bytes(n->x_dtype, shift) * ((pre ? 1 : 0) + (dout ? 1 : 0)) +
                    piece_bytes(n->y_dtype, shift) * ((post ? 1 : 0) + (pre ? 1 : 0));
  if (!backward_plan(n->rows, n->cols, n->tokens, bytes, shift, s, p, blocks))
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
  a.totals_shared = totals_in_shared(s, n->rows, n->tokens);
  a.depth = p.depth; a.slot_bytes = p.slot_bytes;
  blocks = launch_types(a, n->x_dtype, n->y_dtype, s, NormLaunch{true, post, pre, blocks, s.threads(), p.smem, stream});
  if (blocks == 0) return (int)cudaErrorInvalidValue;
  const int rc = (int)cudaGetLastError();
  if (rc != 0 || !(shared || per_sample)) return rc;
  t.rows = n->rows; t.cols = n->cols; t.tokens = n->tokens;
  t.blocks = shared ? blocks : 0;
  t.units = std::min((long long)blocks * s.groups, (long long)n->rows);
  t.sums = a.sums; t.parked = a.parked;
  const long long samples = n->rows / n->tokens;
  t.by_sample = samples < t.units;
  const long long places = per_sample ? std::min(samples, t.units - 1) : 0;
  const long long sets = (places + 1) / 2 + (shared ? 1 : 0);
  if (sets == 0) return 0;
  // launched while the backward kernel's last blocks run: its blocks find their sums and read the vectors until then
  launch_early(norm_sums_kernel, dim3((unsigned)sets, (n->cols + 127) / 128, 2), 512, 0, stream, t);
  return (int)cudaGetLastError();
}
