// Layer norm and its gradients.
//
// Of a row x of D numbers, with m = mean(x), r = (mean((x - m)^2) + eps)^(-1/2):
//   h = (x - m) r,  y = h w + b
// and backward, with u = g w:
//   dx = r (u - mean(u) - h mean(u h)),  dw = sum over rows of g h,  db = sum of g.
#include <hip/hip_runtime.h>

namespace {

constexpr int kThreads = 256;

// The sum over a workgroup, in every thread.
__device__ inline float block_sum(float x) {
  __shared__ float part[kThreads / 64];
#pragma unroll
  for (int d = 32; d > 0; d /= 2) x += __shfl_xor(x, d);
  __syncthreads();
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = x;
  __syncthreads();
  x = 0.f;
#pragma unroll
  for (int i = 0; i < kThreads / 64; i++) x += part[i];
  return x;
}

struct Moments {
  float mean, inv;
};

__device__ inline Moments moments(const float* x, int dim, float eps) {
  float s = 0.f;
  for (int c = threadIdx.x; c < dim; c += kThreads) s += x[c];
  const float mean = block_sum(s) / dim;
  s = 0.f;
  for (int c = threadIdx.x; c < dim; c += kThreads) s += (x[c] - mean) * (x[c] - mean);
  return {mean, 1.f / sqrtf(block_sum(s) / dim + eps)};
}

}  // namespace

extern "C" __global__ void __launch_bounds__(kThreads)
    fg_layer_norm(float* out, const float* x, const float* w, const float* b, int rows, int dim, float eps) {
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const float* row = x + static_cast<size_t>(r) * dim;
    const Moments m = moments(row, dim, eps);
    for (int c = threadIdx.x; c < dim; c += kThreads)
      out[static_cast<size_t>(r) * dim + c] = (row[c] - m.mean) * m.inv * w[c] + (b ? b[c] : 0.f);
  }
}

extern "C" __global__ void __launch_bounds__(kThreads)
    fg_layer_norm_grad(float* dx, const float* x, const float* w, const float* g, float* dw, float* db, float* stats,
                       int rows, int dim, float eps) {
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const size_t at = static_cast<size_t>(r) * dim;
    const Moments m = moments(x + at, dim, eps);
    float su = 0.f, sh = 0.f;
    for (int c = threadIdx.x; c < dim; c += kThreads) {
      const float u = g[at + c] * w[c];
      su += u;
      sh += u * ((x[at + c] - m.mean) * m.inv);
    }
    su = block_sum(su) / dim;
    sh = block_sum(sh) / dim;
    for (int c = threadIdx.x; c < dim; c += kThreads)
      dx[at + c] = m.inv * (g[at + c] * w[c] - su - (x[at + c] - m.mean) * m.inv * sh);
    if (threadIdx.x == 0) {
      stats[2 * static_cast<size_t>(r)] = m.mean;
      stats[2 * static_cast<size_t>(r) + 1] = m.inv;
    }
  }
}

// A thread sums a column.
extern "C" __global__ void __launch_bounds__(kThreads)
    fg_layer_norm_weight(float* dx, const float* x, const float* w, const float* g, float* dw, float* db, float* stats,
                         int rows, int dim, float eps) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= dim) return;
  float sw = 0.f, sb = 0.f;
  for (int r = 0; r < rows; r++) {
    const size_t at = static_cast<size_t>(r) * dim + c;
    sw += g[at] * ((x[at] - stats[2 * static_cast<size_t>(r)]) * stats[2 * static_cast<size_t>(r) + 1]);
    sb += g[at];
  }
  dw[c] = sw;
  if (db) db[c] = sb;
}
