// Rows of an embedding by token, scaled, and the weight's gradient.
//
//   y_t = s W[id_t],  dW_v = s sum over the tokens t with id_t = v of g_t,
// in the order of t. An id outside of [0, vocab) is no token: its row is of
// zeros, and it has no gradient.
#include <hip/hip_runtime.h>

namespace {

constexpr int kThreads = 256;

}  // namespace

extern "C" __global__ void __launch_bounds__(kThreads)
    fg_embedding(float* out, const float* weight, const int* ids, int tokens, int vocab, int dim, float scale) {
  for (int t = blockIdx.x; t < tokens; t += gridDim.x) {
    const int id = ids[t];
    const bool inside = id >= 0 && id < vocab;
    const float* from = weight + static_cast<size_t>(inside ? id : 0) * dim;
    float* to = out + static_cast<size_t>(t) * dim;
    for (int c = threadIdx.x; c < dim; c += kThreads) to[c] = inside ? from[c] * scale : 0.f;
  }
}

// A workgroup goes through all ids for each of its rows.
extern "C" __global__ void __launch_bounds__(kThreads)
    fg_embedding_grad(float* dw, const int* ids, const float* g, int tokens, int vocab, int dim, float scale) {
  const int lane = threadIdx.x % 64;
  for (int v = blockIdx.x; v < vocab; v += gridDim.x)
    for (int c0 = 0; c0 < dim; c0 += kThreads) {
      const int c = c0 + threadIdx.x;
      float sum = 0.f;
      for (int t0 = 0; t0 < tokens; t0 += 64) {
        unsigned long long mine = __ballot(t0 + lane < tokens && ids[min(t0 + lane, tokens - 1)] == v);
        for (; mine; mine &= mine - 1)
          if (c < dim) sum += g[static_cast<size_t>(t0 + __ffsll(mine) - 1) * dim + c];
      }
      if (c < dim) dw[static_cast<size_t>(v) * dim + c] = sum * scale;
    }
}
