// Cross-entropy of token labels, and the logits' gradient.
//
// Of n rows x of C logits with a label each, N of which are in [0, C) (the
// others are ignored):
//   loss = 1/N sum over the N rows of logsumexp(x) - x[label]   (0 if N is 0)
//   dx = g/N (softmax(x) - onehot(label)), 0 in ignored rows.
//
// Bound by memory: the loss reads a row once, the gradient reads and writes it
// once. So a row of up to 65536 logits lives in the registers of L lanes, K
// vectors of four each, from its maximum to its gradient; a longer one is read
// once with a running maximum and sum, and again for its gradient, out of the
// Infinity Cache. A gradient whose g is 1 makes the loss as well: a training step
// reads its logits once. Ignored rows of more than 1024 logits are not read.
//
// 8192 rows of 32000, a tenth ignored, loss and gradient: 363 us (5.5 TB/s; 396
// with the library's exp2, 389 with registers for two workgroups a compute unit,
// 397 with the next row's loads behind this one's stores, which they then wait for).
// 2047 of 50001, a fifth ignored: 148 (5.0 TB/s: a row fills a compute unit, so
// its loads, sums and stores take turns; 176 read twice). Read twice, 8192 of 32000
// take 403. In 16 vectors a lane, whole rows leave 16 bytes a lane in scratch
// memory.
#include <hip/hip_runtime.h>

#include "rows.hpp"

namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

// 2^x by the hardware's instruction alone: within a step, and 0 below the normal
// range, where the library's function scales twice. Here 0 stands for what is
// below 2^-126 of a sum that is 1 or more. Its argument, (x - top) log2(e), is one
// rounded product of a rounded constant: e^-d is off by up to 1.2 d half steps
// besides, 37 of a probability of 1e-13, which is as little of a sum as its small
// terms are.
__device__ inline float power2(float x) { return __builtin_amdgcn_exp2f(x); }

// Sum of whole numbers or of doubles over a workgroup, in every thread.
template <int THREADS, class T>
__device__ inline T block_sum(T x) {
  __shared__ T part[THREADS / 64];
#pragma unroll
  for (int d = 32; d > 0; d /= 2) x += __shfl_xor(x, d);
  __syncthreads();
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = x;
  __syncthreads();
  x = part[0];
#pragma unroll
  for (int i = 1; i < THREADS / 64; i++) x += part[i];
  return x;
}

__device__ inline bool is_class(int label, int classes) { return label >= 0 && label < classes; }

// How many of the labels are classes: those of a workgroup's part of the rows, and
// of all of them: the sum of what a launch of kParts workgroups counted, or, without
// it, counted by each workgroup for itself.
constexpr int kParts = 16;
template <int THREADS>
__device__ inline int count_valid(const int* __restrict__ labels, int rows, int classes, unsigned part, unsigned parts) {
  int n = 0;
#pragma unroll 8
  for (int r = part * THREADS + threadIdx.x; r < rows; r += parts * THREADS) n += is_class(labels[r], classes);
  return block_sum<THREADS>(n);
}
template <int THREADS>
__device__ inline int all_valid(const int* __restrict__ counts, const int* __restrict__ labels, int rows, int classes) {
  if (!counts) return count_valid<THREADS>(labels, rows, classes, 0, 1);
  int n = 0;
#pragma unroll
  for (int i = 0; i < kParts; i++) n += counts[i];
  return n;
}

// A part of the loss: the sum of losses of some rows, and how many of them are
// valid, by one thread. The only one makes the mean; others are left to a launch of
// one workgroup.
__device__ inline void give_loss(float* loss, float* sums, int* valid, int at, double s, int n) {
  if (gridDim.x == 1) {
    *loss = static_cast<float>(s / max(n, 1));
  } else {
    // A rounding of a sum of losses, which are rounded themselves.
    sums[at] = static_cast<float>(s);
    valid[at] = n;
  }
}
template <int THREADS>
__device__ inline void mean_loss(float* loss, const float* __restrict__ sums, const int* __restrict__ valid, int parts) {
  int n = 0;
  double s = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < parts; i += THREADS) {
    n += valid[i];
    s += sums[i];
  }
  n = block_sum<THREADS>(n);
  s = block_sum<THREADS>(s);
  if (threadIdx.x == 0) *loss = static_cast<float>(s / max(n, 1));
}

constexpr int kLine = 32;  // floats

// A row's loss: its label's logit, its largest one, and the sum of exp(x - top).
__device__ inline float row_loss(float picked, float top, float sum) { return (top - picked) + log2f(sum) * kLn2; }

// Rows on L lanes each: the loss where `sums` is not null; with `Grad` dx, their
// gradients, g (or null: 1) over the number of valid labels times what it says
// above.
template <int L, int K, bool Whole, bool Grad, bool Stream>
__device__ inline void rows_of(float* __restrict__ dx, const float* __restrict__ x, const int* __restrict__ labels,
                               const float* __restrict__ g, const int* __restrict__ counts, float* __restrict__ loss,
                               float* __restrict__ sums, int* __restrict__ valids, int rows, int classes) {
  constexpr int kThreads = threads_of(L), kGroups = kThreads / L;
  Columns<L, K, Whole> cols(classes);
  // Rounded once for all of the gradient, where a division of each element would
  // round each by itself.
  float scale = 0.f;
  if (Grad) scale = (g ? *g : 1.f) / max(all_valid<kThreads>(counts, labels, rows, classes), 1);
  double total = 0.0;
  int in = 0;
  for (int r0 = blockIdx.x * kGroups; r0 < rows; r0 += gridDim.x * kGroups) {
    const int r = r0 + static_cast<int>(threadIdx.x) / L, label = labels[min(r, rows - 1)];
    const bool valid = is_class(label, classes);
    const size_t at = static_cast<size_t>(min(r, rows - 1)) * classes;
    // Long rows begin on cache lines, whatever their width: 2047 of 50001 148 us,
    // not 158; 8192 of 4001 would take 45.4, not 44.5. So equal rows that begin
    // elsewhere in their lines are added up in other orders.
    if (!Whole && L * K >= 2048) cols.from = -static_cast<int>(at % kLine);
    Vec<4> v[K];
    if (L > 64 && !valid) {  // the same in all of the workgroup
      if (sums && threadIdx.x == 0) give_loss(loss, sums, valids, r, 0.0, 0);
      if (Grad)
#pragma unroll
        for (int k = 0; k < K; k++) cols.template write<Stream>(dx + at, k, Vec<4>{});
      continue;
    }
    const float picked = x[at + (valid ? label : 0)];
    cols.template read<Stream>(v, x + at, -INFINITY);
    float top[1] = {-INFINITY}, sum[1] = {};
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int e = 0; e < 4; e++) top[0] = fmaxf(top[0], v[k].v[e]);
    join_row<L>(top, Largest());
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        v[k].v[e] = power2((v[k].v[e] - top[0]) * kLog2e);
        sum[0] += v[k].v[e];
      }
    row_sums<L>(sum);
    if (r >= rows) continue;
    // Of long rows each is a part, of others those of a workgroup.
    if (L > 64) {
      if (sums && threadIdx.x == 0) give_loss(loss, sums, valids, r, row_loss(picked, top[0], sum[0]), 1);
    } else if (cols.lane == 0 && valid) {
      total += row_loss(picked, top[0], sum[0]);
      in++;
    }
    if (!Grad) continue;
    const float inv = 1.f / sum[0];
#pragma unroll
    for (int k = 0; k < K; k++) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float p = v[k].v[e] * inv - (cols.at(k) + e == label ? 1.f : 0.f);
        v[k].v[e] = valid ? p * scale : 0.f;
      }
      cols.template write<Stream>(dx + at, k, v[k]);
    }
  }
  if (L > 64 || !sums) return;
  total = block_sum<kThreads>(total);
  in = block_sum<kThreads>(in);
  if (threadIdx.x == 0) give_loss(loss, sums, valids, blockIdx.x, total, in);
}

// ── rows of more than registers hold ────────────────────────────────────────

constexpr int kLong = 1024;  // threads
constexpr int kBatch = 8;    // vectors of a thread on their way at a time

// f(first column, up to four logits) over the row, a thread's vectors in batches.
template <bool Stream, class F>
__device__ inline void over_row(const float* __restrict__ row, int classes, F f) {
  for (int c0 = 0; c0 < classes; c0 += kBatch * kLong * 4) {
    Vec<4> v[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; k++) {
      const int c = c0 + (k * kLong + static_cast<int>(threadIdx.x)) * 4;
      if (c + 4 <= classes) {
        v[k] = load<4, Stream>(row + c);
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) v[k].v[e] = c + e < classes ? row[c + e] : -INFINITY;
      }
    }
    f(c0, v);
  }
}

template <bool Grad>
__device__ inline void long_rows(float* __restrict__ dx, const float* __restrict__ x, const int* __restrict__ labels,
                                 const float* __restrict__ g, const int* __restrict__ counts, float* __restrict__ loss,
                                 float* __restrict__ sums, int* __restrict__ valids, int rows, int classes) {
  float scale = 0.f;
  if (Grad) scale = (g ? *g : 1.f) / max(all_valid<kLong>(counts, labels, rows, classes), 1);
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const int label = labels[r];
    const size_t at = static_cast<size_t>(r) * classes;
    if (!is_class(label, classes)) {
      if (sums && threadIdx.x == 0) give_loss(loss, sums, valids, r, 0.0, 0);
      if (Grad)
        for (int c = threadIdx.x; c < classes; c += kLong) dx[at + c] = 0.f;
      continue;
    }
    const float picked = x[at + label];
    // A running maximum, and the sum of exp(x - it). While all are -inf the sum
    // is of exp(x): 0.
    float top[1] = {-INFINITY}, sum[1] = {};
    over_row<false>(x + at, classes, [&](int, Vec<4>(&v)[kBatch]) {
      float now = top[0];
#pragma unroll
      for (int k = 0; k < kBatch; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) now = fmaxf(now, v[k].v[e]);
      const float from = now == -INFINITY ? 0.f : now;
      sum[0] *= power2((top[0] - from) * kLog2e);
      top[0] = now;
#pragma unroll
      for (int k = 0; k < kBatch; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) sum[0] += power2((v[k].v[e] - from) * kLog2e);
    });
    const float mine = top[0];
    join_row<kLong>(top, Largest());
    sum[0] *= power2((mine - (top[0] == -INFINITY ? 0.f : top[0])) * kLog2e);
    row_sums<kLong>(sum);
    if (sums && threadIdx.x == 0) give_loss(loss, sums, valids, r, row_loss(picked, top[0], sum[0]), 1);
    if (!Grad) continue;
    const float inv = 1.f / sum[0], from = top[0];
    over_row<false>(x + at, classes, [&](int c0, Vec<4>(&v)[kBatch]) {
#pragma unroll
      for (int k = 0; k < kBatch; k++) {
        const int c = c0 + (k * kLong + static_cast<int>(threadIdx.x)) * 4;
#pragma unroll
        for (int e = 0; e < 4; e++)
          v[k].v[e] = (power2((v[k].v[e] - from) * kLog2e) * inv - (c + e == label ? 1.f : 0.f)) * scale;
        if (c + 4 <= classes) {
          store<4, true>(dx + at + c, v[k]);
        } else {
#pragma unroll
          for (int e = 0; e < 3; e++)
            if (c + e < classes) dx[at + c + e] = v[k].v[e];
        }
      }
    });
  }
}

}  // namespace

// The first output is the loss of a forward call, dx of a gradient.
#define FG_LOSS_ARGS \
  float *loss, const float *x, const int *labels, float *sums, int *valids, int parts, int rows, int classes
#define FG_GRAD_ARGS                                                                                                    \
  float *dx, const float *x, const int *labels, const float *g, float *loss, float *sums, int *valids, int parts,       \
      int *counts, int rows, int classes

#define FG_LOSS_AS(L, K, NAME, WHOLE)                                                                                     \
  extern "C" __global__ void __launch_bounds__(threads_of(L)) fg_token_loss_##NAME(FG_LOSS_ARGS) {                        \
    rows_of<L, K, WHOLE, false, false>(nullptr, x, labels, nullptr, nullptr, loss, sums, valids, rows, classes);       \
  }
#define FG_GRAD_AS(L, K, NAME, WHOLE, STREAM)                                                                             \
  extern "C" __global__ void __launch_bounds__(threads_of(L)) fg_token_loss_grad_##NAME(FG_GRAD_ARGS) {                   \
    rows_of<L, K, WHOLE, true, STREAM>(dx, x, labels, g, counts, loss, sums, valids, rows, classes);               \
  }
#define FG_TOKEN_LOSS(L, K)                             \
  FG_LOSS_AS(L, K, L##_##K, true)                       \
  FG_LOSS_AS(L, K, L##_##K##_odd, false)                \
  FG_GRAD_AS(L, K, L##_##K, true, false)                \
  FG_GRAD_AS(L, K, L##_##K##_stream, true, true)        \
  FG_GRAD_AS(L, K, L##_##K##_odd, false, false)         \
  FG_GRAD_AS(L, K, L##_##K##_odd_stream, false, true)

FG_TOKEN_LOSS(8, 1)
FG_TOKEN_LOSS(16, 1)
FG_TOKEN_LOSS(32, 1)
FG_TOKEN_LOSS(64, 1)
FG_TOKEN_LOSS(64, 2)
FG_TOKEN_LOSS(64, 4)
FG_TOKEN_LOSS(256, 2)
FG_TOKEN_LOSS(256, 4)
FG_TOKEN_LOSS(256, 8)
FG_TOKEN_LOSS(512, 8)
FG_TOKEN_LOSS(1024, 8)
FG_TOKEN_LOSS(1024, 16)

extern "C" __global__ void __launch_bounds__(kLong) fg_token_loss_long(FG_LOSS_ARGS) {
  long_rows<false>(nullptr, x, labels, nullptr, nullptr, loss, sums, valids, rows, classes);
}
extern "C" __global__ void __launch_bounds__(kLong) fg_token_loss_grad_long(FG_GRAD_ARGS) {
  long_rows<true>(dx, x, labels, g, counts, loss, sums, valids, rows, classes);
}

extern "C" __global__ void __launch_bounds__(kLong) fg_token_loss_mean(FG_LOSS_ARGS) {
  mean_loss<kLong>(loss, sums, valids, parts);
}
extern "C" __global__ void __launch_bounds__(kLong) fg_token_loss_grad_mean(FG_GRAD_ARGS) {
  mean_loss<kLong>(loss, sums, valids, parts);
}
extern "C" __global__ void __launch_bounds__(kLong) fg_token_loss_grad_count(FG_GRAD_ARGS) {
  const int n = count_valid<kLong>(labels, rows, classes, blockIdx.x, gridDim.x);
  if (threadIdx.x == 0) counts[blockIdx.x] = n;
}
