// Attention and its gradients.
//
//   S_ij = scale q_i . k_j over the keys j that query i sees, y_i = softmax(S_i) v
// Query head h of batch b reads key head h / (Hq / Hk). Keys at or past
// lengths[b] are hidden, and with `causal` those past i + Sk - Sq. A query that
// sees no key gives 0 and gradients of 0.
// Matrices are one row per token: q, y [B Sq, Hq D], k, v [B Sk, Hk D].
// stats holds per (b, h, i) the row's maximum in units of log2 (of S log2 e),
// then 1 / sum, for the gradients to make the probabilities again.
#include <hip/hip_runtime.h>

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

struct Shape {
  int b, sq, sk, hq, hk, d, causal;
};

// Keys of batch b.
__device__ inline int key_count(const Shape& s, const int* lengths, int b) {
  return lengths ? min(max(lengths[b], 0), s.sk) : s.sk;
}

// Keys that query i sees: those below this.
__device__ inline int visible(const Shape& s, int keys, int i) {
  return s.causal ? max(0, min(keys, i + s.sk - s.sq + 1)) : keys;
}

__device__ inline float wave_max(float x) {
  for (int d = 32; d > 0; d /= 2) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}
__device__ inline float wave_sum(float x) {
  for (int d = 32; d > 0; d /= 2) x += __shfl_xor(x, d);
  return x;
}

__device__ inline float dot(const float* a, const float* b, int d) {
  float t = 0.f;
  for (int e = 0; e < d; e++) t += a[e] * b[e];
  return t;
}

}  // namespace

// One wave per query row.
extern "C" __global__ void __launch_bounds__(256)
    fg_attention(float* __restrict__ y, const float* __restrict__ q, const float* __restrict__ k,
                 const float* __restrict__ v, float* __restrict__ stats, const int* __restrict__ lengths, int B, int Sq,
                 int Sk, int Hq, int Hk, int D, int causal, float scale) {
  __shared__ float probs[4][64];
  const Shape s{B, Sq, Sk, Hq, Hk, D, causal};
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const size_t row = static_cast<size_t>(blockIdx.x) * 4 + wave;  // (b, h, i)
  const bool live = row < static_cast<size_t>(B) * Hq * Sq;
  const int i = live ? row % Sq : 0, h = live ? row / Sq % Hq : 0, b = live ? row / Sq / Hq : 0;
  const int hk = h / (Hq / Hk);
  const int seen = live ? visible(s, key_count(s, lengths, b), i) : 0;
  const float* qi = q + (static_cast<size_t>(b) * Sq + i) * Hq * D + static_cast<size_t>(h) * D;
  const float* kb = k + static_cast<size_t>(b) * Sk * Hk * D + static_cast<size_t>(hk) * D;
  const float* vb = v + static_cast<size_t>(b) * Sk * Hk * D + static_cast<size_t>(hk) * D;
  const size_t stride = static_cast<size_t>(Hk) * D;
  float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
  for (int j0 = 0; j0 < seen; j0 += 64) {
    const int j = j0 + lane;
    const float x = j < seen ? dot(qi, kb + j * stride, D) * (scale * kLog2e) : -INFINITY;
    const float top = fmaxf(m, wave_max(x)), base = top == -INFINITY ? 0.f : top;
    const float p = exp2f(x - base), old = exp2f(m - base);
    l = l * old + wave_sum(p);
    m = top;
    probs[wave][lane] = p;
    __builtin_amdgcn_wave_barrier();
    for (int t = 0; t < 2; t++) {
      const int d = lane + 64 * t;
      if (d >= D) continue;
      float sum = 0.f;
      for (int n = 0; n < min(64, seen - j0); n++) sum += probs[wave][n] * vb[(j0 + n) * stride + d];
      o[t] = o[t] * old + sum;
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (!live) return;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  for (int t = 0; t < 2; t++)
    if (lane + 64 * t < D) y[(static_cast<size_t>(b) * Sq + i) * Hq * D + static_cast<size_t>(h) * D + lane + 64 * t] = o[t] * inv;
  if (lane == 0) {
    stats[row] = m == -INFINITY ? 0.f : m;
    stats[static_cast<size_t>(B) * Hq * Sq + row] = inv;
  }
}

// dq: one wave per query row.
extern "C" __global__ void __launch_bounds__(256)
    fg_attention_dq(float* __restrict__ dq, const float* __restrict__ q, const float* __restrict__ k,
                    const float* __restrict__ v, const float* __restrict__ y, const float* __restrict__ g,
                    const float* __restrict__ stats, float* __restrict__ dk, float* __restrict__ dv,
                    const int* __restrict__ lengths, int B, int Sq, int Sk, int Hq, int Hk, int D, int causal,
                    float scale) {
  __shared__ float probs[4][64];
  const Shape s{B, Sq, Sk, Hq, Hk, D, causal};
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const size_t rows = static_cast<size_t>(B) * Hq * Sq, row = static_cast<size_t>(blockIdx.x) * 4 + wave;
  const bool live = row < rows;
  const int i = live ? row % Sq : 0, h = live ? row / Sq % Hq : 0, b = live ? row / Sq / Hq : 0;
  const int hk = h / (Hq / Hk);
  const int seen = live ? visible(s, key_count(s, lengths, b), i) : 0;
  const size_t at = (static_cast<size_t>(b) * Sq + i) * Hq * D + static_cast<size_t>(h) * D;
  const float* kb = k + static_cast<size_t>(b) * Sk * Hk * D + static_cast<size_t>(hk) * D;
  const float* vb = v + static_cast<size_t>(b) * Sk * Hk * D + static_cast<size_t>(hk) * D;
  const size_t stride = static_cast<size_t>(Hk) * D;
  const float m = live ? stats[row] : 0.f, inv = live ? stats[rows + row] : 0.f;
  const float delta = dot(g + at, y + at, D);
  float o[2] = {0.f, 0.f};
  for (int j0 = 0; j0 < seen; j0 += 64) {
    const int j = j0 + lane;
    float ds = 0.f;
    if (j < seen) {
      const float p = exp2f(dot(q + at, kb + j * stride, D) * (scale * kLog2e) - m) * inv;
      ds = p * (dot(g + at, vb + j * stride, D) - delta) * scale;
    }
    probs[wave][lane] = ds;
    __builtin_amdgcn_wave_barrier();
    for (int t = 0; t < 2; t++) {
      const int d = lane + 64 * t;
      if (d >= D) continue;
      for (int n = 0; n < min(64, seen - j0); n++) o[t] += probs[wave][n] * kb[(j0 + n) * stride + d];
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (!live) return;
  for (int t = 0; t < 2; t++)
    if (lane + 64 * t < D) dq[at + lane + 64 * t] = o[t];
}

// dk, dv: one wave per key row, over the queries of every head that reads it.
extern "C" __global__ void __launch_bounds__(256)
    fg_attention_dkv(float* __restrict__ dq, const float* __restrict__ q, const float* __restrict__ k,
                     const float* __restrict__ v, const float* __restrict__ y, const float* __restrict__ g,
                     const float* __restrict__ stats, float* __restrict__ dk, float* __restrict__ dv,
                     const int* __restrict__ lengths, int B, int Sq, int Sk, int Hq, int Hk, int D, int causal,
                     float scale) {
  __shared__ float probs[4][64], grads[4][64];
  const Shape s{B, Sq, Sk, Hq, Hk, D, causal};
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const size_t rows = static_cast<size_t>(B) * Hq * Sq, row = static_cast<size_t>(blockIdx.x) * 4 + wave;
  if (row >= static_cast<size_t>(B) * Hk * Sk) return;
  const int j = row % Sk, hk = row / Sk % Hk, b = row / Sk / Hk;
  const int keys = key_count(s, lengths, b), group = Hq / Hk;
  const size_t at = (static_cast<size_t>(b) * Sk + j) * Hk * D + static_cast<size_t>(hk) * D;
  const size_t stride = static_cast<size_t>(Hq) * D;
  float ok[2] = {0.f, 0.f}, ov[2] = {0.f, 0.f};
  const int first = causal ? max(0, j - (Sk - Sq)) : 0;
  for (int h = hk * group; h < (hk + 1) * group && j < keys; h++) {
    const size_t base = static_cast<size_t>(b) * Sq * Hq * D + static_cast<size_t>(h) * D;
    const float* st = stats + (static_cast<size_t>(b) * Hq + h) * Sq;
    for (int i0 = first; i0 < Sq; i0 += 64) {
      const int i = i0 + lane;
      float p = 0.f, ds = 0.f;
      if (i < Sq) {
        const size_t qi = base + i * stride;
        p = exp2f(dot(q + qi, k + at, D) * (scale * kLog2e) - st[i]) * st[rows + i];
        ds = p * (dot(g + qi, v + at, D) - dot(g + qi, y + qi, D)) * scale;
      }
      probs[wave][lane] = p;
      grads[wave][lane] = ds;
      __builtin_amdgcn_wave_barrier();
      for (int t = 0; t < 2; t++) {
        const int d = lane + 64 * t;
        if (d >= D) continue;
        for (int n = 0; n < min(64, Sq - i0); n++) {
          ov[t] += probs[wave][n] * g[base + (i0 + n) * stride + d];
          ok[t] += grads[wave][n] * q[base + (i0 + n) * stride + d];
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
  for (int t = 0; t < 2; t++)
    if (lane + 64 * t < D) {
      dk[at + lane + 64 * t] = ok[t];
      dv[at + lane + 64 * t] = ov[t];
    }
}
