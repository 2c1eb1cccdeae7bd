// Cross-entropy of token labels, and the logits' gradient.
//
// Of n rows x of C logits with a label each, N of which are in [0, C) (the
// others are ignored):
//   loss = 1/N sum over the N rows of logsumexp(x) - x[label]   (0 if N is 0)
//   dx = g/N (softmax(x) - onehot(label)), 0 in ignored rows.
#include <hip/hip_runtime.h>

namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

template <class T, class F>
__device__ inline T block_all(T x, F join) {
  __shared__ T part[kThreads / 64];
#pragma unroll
  for (int d = 32; d > 0; d /= 2) x = join(x, __shfl_xor(x, d));
  __syncthreads();
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = x;
  __syncthreads();
  x = part[0];
#pragma unroll
  for (int i = 1; i < kThreads / 64; i++) x = join(x, part[i]);
  return x;
}

template <class T>
__device__ inline T block_sum(T x) {
  return block_all(x, [](T a, T b) { return a + b; });
}

struct Row {
  float top, sum;  // the largest logit, and the sum of exp(x - top)
};

__device__ inline Row row_sum(const float* x, int classes) {
  // NaN is kept: fmaxf would drop it, but the sum below has it.
  float top = -INFINITY;
  for (int c = threadIdx.x; c < classes; c += kThreads) top = fmaxf(top, x[c]);
  top = block_all(top, [](float a, float b) { return fmaxf(a, b); });
  float s = 0.f;
  for (int c = threadIdx.x; c < classes; c += kThreads) s += exp2f((x[c] - top) * kLog2e);
  return {top, block_sum(s)};
}

__device__ inline int count_valid(const int* labels, int rows, int classes) {
  int n = 0;
  for (int r = threadIdx.x; r < rows; r += kThreads) n += labels[r] >= 0 && labels[r] < classes;
  return block_sum(n);
}

}  // namespace

extern "C" __global__ void __launch_bounds__(kThreads)
    fg_token_loss(float* out, const float* x, const int* labels, float* each, int rows, int classes) {
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const int label = labels[r];
    float v = 0.f;
    if (label >= 0 && label < classes) {
      const float* row = x + static_cast<size_t>(r) * classes;
      const Row s = row_sum(row, classes);
      v = (s.top - row[label]) + log2f(s.sum) * kLn2;
    }
    if (threadIdx.x == 0) each[r] = v;
  }
}

extern "C" __global__ void __launch_bounds__(kThreads)
    fg_token_loss_mean(float* out, const float* x, const int* labels, float* each, int rows, int classes) {
  const int n = count_valid(labels, rows, classes);
  double s = 0.0;
  for (int r = threadIdx.x; r < rows; r += kThreads) s += each[r];
  s = block_sum(s);
  if (threadIdx.x == 0) *out = static_cast<float>(s / max(n, 1));
}

extern "C" __global__ void __launch_bounds__(kThreads)
    fg_token_loss_grad(float* dx, const float* x, const int* labels, const float* g, int rows, int classes) {
  const float scale = *g / max(count_valid(labels, rows, classes), 1);
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const int label = labels[r];
    const size_t at = static_cast<size_t>(r) * classes;
    if (label >= 0 && label < classes) {
      const Row s = row_sum(x + at, classes);
      const float inv = 1.f / s.sum;
      for (int c = threadIdx.x; c < classes; c += kThreads)
        dx[at + c] = (exp2f((x[at + c] - s.top) * kLog2e) * inv - (c == label ? 1.f : 0.f)) * scale;
    } else {
      for (int c = threadIdx.x; c < classes; c += kThreads) dx[at + c] = 0.f;
    }
  }
}
