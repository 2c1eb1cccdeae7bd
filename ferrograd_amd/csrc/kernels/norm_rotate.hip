// Norms of each head with the position rotation in the same pass, and their
// gradients.
//
// A row is one head of one token, D numbers x:
//   r = (mean(x^2) + eps)^(-1/2),  z = x r w,
//   (y_i, y_{i + D/2}) = (z_i cos - z_{i + D/2} sin, z_{i + D/2} cos + z_i sin)
// with the angle pos * base^(-2i/D), i < D/2. Backward, with g' the gradient
// rotated back and n = x r:
//   dx = r (g' w - n mean(g' w n)),  dw = sum over rows of g' n.
//
// Bound by memory: forward reads and writes a row once (8 bytes an element),
// backward reads x and g and writes dx (12). So a row lives in the registers
// of G lanes (the least power of two that holds half a row in vectors of VEC,
// so lane i has both numbers of its pairs), its sums run over the G lanes, and
// the cosines of a token are made once and serve several of its heads. Angles
// are formed in 64 bits as revolutions and reduced there: a far position times
// a frequency has more whole turns than 32 bits can hold beside the fraction.
// dw is summed in registers over all rows of a group, then over the workgroup
// in LDS, then over the workgroups by a second launch: a fixed order, no
// atomics.
#include <hip/hip_runtime.h>

namespace {

constexpr int kThreads = 256;

template <int VEC>
struct Vec {
  float v[VEC];
};

template <int VEC>
__device__ inline Vec<VEC> load(const float* p) {
  Vec<VEC> r;
  if constexpr (VEC == 4) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    r = {{t.x, t.y, t.z, t.w}};
  } else if constexpr (VEC == 2) {
    const float2 t = *reinterpret_cast<const float2*>(p);
    r = {{t.x, t.y}};
  } else {
    r.v[0] = *p;
  }
  return r;
}

template <int VEC>
__device__ inline void store(float* p, const Vec<VEC>& r) {
  if constexpr (VEC == 4) *reinterpret_cast<float4*>(p) = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
  else if constexpr (VEC == 2) *reinterpret_cast<float2*>(p) = make_float2(r.v[0], r.v[1]);
  else *p = r.v[0];
}

template <int G>
__device__ inline float group_sum(float x) {
#pragma unroll
  for (int d = G / 2; d > 0; d /= 2) x += __shfl_xor(x, d, G);
  return x;
}

// The frequencies (revolutions per position) of a lane's pairs.
template <int VEC, int G, int NV>
__device__ inline void frequencies(double (&freq)[NV][VEC], int sub, int half, double log2_base) {
#pragma unroll
  for (int v = 0; v < NV; v++)
#pragma unroll
    for (int e = 0; e < VEC; e++) {
      const int i = (v * G + sub) * VEC + e;
      freq[v][e] = exp2(-(static_cast<double>(i) / half) * log2_base) * 0.15915494309189533577;  // 1 / (2 pi)
    }
}

// cos and sin of pos * frequency; the whole turns go in 64 bits.
__device__ inline void turn(double freq, int pos, float* c, float* s) {
  const double t = freq * pos;
  sincospif(2.f * static_cast<float>(t - rint(t)), s, c);
}

// Units of work: `heads_per` heads of a token; group g of the launch takes
// units g, g + groups, ...
template <int VEC, int G, int NV>
__device__ inline void forward(float* __restrict__ out, const float* __restrict__ x, const float* __restrict__ w,
                               const int* __restrict__ positions, int tokens, int heads, int dim, int heads_per,
                               float eps, float log2_base_hi, float log2_base_lo) {
  const int half = dim / 2, sub = threadIdx.x % G;
  const unsigned groups = gridDim.x * (kThreads / G);
  const unsigned chunks = (heads + heads_per - 1) / heads_per;
  const unsigned units = static_cast<unsigned>(tokens) * chunks;
  double freq[NV][VEC];
  frequencies<VEC, G, NV>(freq, sub, half, static_cast<double>(log2_base_hi) + log2_base_lo);
  Vec<VEC> wa[NV], wb[NV];
#pragma unroll
  for (int v = 0; v < NV; v++) {
    const int i = (v * G + sub) * VEC;
    if (i < half) {
      wa[v] = load<VEC>(w + i);
      wb[v] = load<VEC>(w + half + i);
    }
  }
  for (unsigned u = blockIdx.x * (kThreads / G) + threadIdx.x / G; u < units; u += groups) {
    const unsigned token = u / chunks;
    const int h0 = static_cast<int>(u % chunks) * heads_per, h1 = min(heads, h0 + heads_per);
    const int pos = positions[token];
    float c[NV][VEC], s[NV][VEC];
#pragma unroll
    for (int v = 0; v < NV; v++)
#pragma unroll
      for (int e = 0; e < VEC; e++) turn(freq[v][e], pos, &c[v][e], &s[v][e]);
    size_t row = (static_cast<size_t>(token) * heads + h0) * dim;
    for (int h = h0; h < h1; h++, row += dim) {
      Vec<VEC> a[NV], b[NV];
      float ss = 0.f;
#pragma unroll
      for (int v = 0; v < NV; v++) {
        const int i = (v * G + sub) * VEC;
        if (i < half) {
          a[v] = load<VEC>(x + row + i);
          b[v] = load<VEC>(x + row + half + i);
#pragma unroll
          for (int e = 0; e < VEC; e++) ss += a[v].v[e] * a[v].v[e] + b[v].v[e] * b[v].v[e];
        }
      }
      const float r = 1.f / sqrtf(group_sum<G>(ss) / dim + eps);
#pragma unroll
      for (int v = 0; v < NV; v++) {
        const int i = (v * G + sub) * VEC;
        if (i >= half) continue;
        Vec<VEC> ya, yb;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const float za = a[v].v[e] * r * wa[v].v[e], zb = b[v].v[e] * r * wb[v].v[e];
          ya.v[e] = za * c[v][e] - zb * s[v][e];
          yb.v[e] = zb * c[v][e] + za * s[v][e];
        }
        store<VEC>(out + row + i, ya);
        store<VEC>(out + row + half + i, yb);
      }
    }
  }
}

template <int VEC, int G, int NV>
__device__ inline void backward(float* __restrict__ dx, const float* __restrict__ x, const float* __restrict__ w,
                                const int* __restrict__ positions, const float* __restrict__ g,
                                float* __restrict__ partial, int tokens, int heads, int dim, int heads_per, float eps,
                                float log2_base_hi, float log2_base_lo) {
  __shared__ float sums[kThreads * 2 * NV * VEC];  // [group of the workgroup][half][index], index < G * NV * VEC
  const int half = dim / 2, sub = threadIdx.x % G, group = threadIdx.x / G;
  const unsigned groups = gridDim.x * (kThreads / G);
  const unsigned chunks = (heads + heads_per - 1) / heads_per;
  const unsigned units = static_cast<unsigned>(tokens) * chunks;
  double freq[NV][VEC];
  frequencies<VEC, G, NV>(freq, sub, half, static_cast<double>(log2_base_hi) + log2_base_lo);
  Vec<VEC> wa[NV], wb[NV];
  float da[NV][VEC] = {}, db[NV][VEC] = {};
#pragma unroll
  for (int v = 0; v < NV; v++) {
    const int i = (v * G + sub) * VEC;
    if (i < half) {
      wa[v] = load<VEC>(w + i);
      wb[v] = load<VEC>(w + half + i);
    }
  }
  for (unsigned u = blockIdx.x * (kThreads / G) + group; u < units; u += groups) {
    const unsigned token = u / chunks;
    const int h0 = static_cast<int>(u % chunks) * heads_per, h1 = min(heads, h0 + heads_per);
    const int pos = positions[token];
    float c[NV][VEC], s[NV][VEC];
#pragma unroll
    for (int v = 0; v < NV; v++)
#pragma unroll
      for (int e = 0; e < VEC; e++) turn(freq[v][e], pos, &c[v][e], &s[v][e]);
    size_t row = (static_cast<size_t>(token) * heads + h0) * dim;
    for (int h = h0; h < h1; h++, row += dim) {
      Vec<VEC> a[NV], b[NV], ga[NV], gb[NV];  // x, and g rotated back
      float ss = 0.f, sg = 0.f;               // sums of x^2 and of g' w x
#pragma unroll
      for (int v = 0; v < NV; v++) {
        const int i = (v * G + sub) * VEC;
        if (i >= half) continue;
        a[v] = load<VEC>(x + row + i);
        b[v] = load<VEC>(x + row + half + i);
        const Vec<VEC> p = load<VEC>(g + row + i), q = load<VEC>(g + row + half + i);
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          ga[v].v[e] = p.v[e] * c[v][e] + q.v[e] * s[v][e];
          gb[v].v[e] = q.v[e] * c[v][e] - p.v[e] * s[v][e];
          ss += a[v].v[e] * a[v].v[e] + b[v].v[e] * b[v].v[e];
          sg += ga[v].v[e] * wa[v].v[e] * a[v].v[e] + gb[v].v[e] * wb[v].v[e] * b[v].v[e];
        }
      }
      const float r = 1.f / sqrtf(group_sum<G>(ss) / dim + eps);
      const float mean = group_sum<G>(sg) * r / dim;
#pragma unroll
      for (int v = 0; v < NV; v++) {
        const int i = (v * G + sub) * VEC;
        if (i >= half) continue;
        Vec<VEC> oa, ob;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const float na = a[v].v[e] * r, nb = b[v].v[e] * r;
          oa.v[e] = r * (ga[v].v[e] * wa[v].v[e] - na * mean);
          ob.v[e] = r * (gb[v].v[e] * wb[v].v[e] - nb * mean);
          da[v][e] += ga[v].v[e] * na;
          db[v][e] += gb[v].v[e] * nb;
        }
        store<VEC>(dx + row + i, oa);
        store<VEC>(dx + row + half + i, ob);
      }
    }
  }
  constexpr int kHalf = G * NV * VEC;
#pragma unroll
  for (int v = 0; v < NV; v++)
#pragma unroll
    for (int e = 0; e < VEC; e++) {
      const int i = (v * G + sub) * VEC + e;
      sums[group * 2 * kHalf + i] = da[v][e];
      sums[group * 2 * kHalf + kHalf + i] = db[v][e];
    }
  __syncthreads();
  for (int d = threadIdx.x; d < dim; d += kThreads) {
    const int at = d < half ? d : kHalf + d - half;
    float t = 0.f;
    for (int k = 0; k < kThreads / G; k++) t += sums[k * 2 * kHalf + at];
    partial[static_cast<size_t>(blockIdx.x) * dim + d] = t;
  }
}

}  // namespace

#define FG_NORM_ROTATE(VEC, G, NV)                                                                                     \
  extern "C" __global__ void __launch_bounds__(kThreads) fg_norm_rotate_##VEC##_##G##_##NV(                            \
      float* out, const float* x, const float* w, const int* positions, int tokens, int heads, int dim, int heads_per, \
      float eps, float log2_base_hi, float log2_base_lo) {                                                             \
    forward<VEC, G, NV>(out, x, w, positions, tokens, heads, dim, heads_per, eps, log2_base_hi, log2_base_lo);         \
  }                                                                                                                    \
  extern "C" __global__ void __launch_bounds__(kThreads) fg_norm_rotate_grad_##VEC##_##G##_##NV(                       \
      float* dx, const float* x, const float* w, const int* positions, const float* g, float* dw, float* partial,      \
      int blocks, int tokens, int heads, int dim, int heads_per, float eps, float log2_base_hi, float log2_base_lo) {  \
    backward<VEC, G, NV>(dx, x, w, positions, g, partial, tokens, heads, dim, heads_per, eps, log2_base_hi,            \
                         log2_base_lo);                                                                                \
  }

FG_NORM_ROTATE(4, 8, 1)
FG_NORM_ROTATE(4, 16, 1)
FG_NORM_ROTATE(4, 32, 1)
FG_NORM_ROTATE(4, 64, 1)
FG_NORM_ROTATE(2, 8, 1)
FG_NORM_ROTATE(2, 16, 1)
FG_NORM_ROTATE(2, 32, 1)
FG_NORM_ROTATE(2, 64, 1)
FG_NORM_ROTATE(2, 64, 2)
FG_NORM_ROTATE(1, 8, 1)
FG_NORM_ROTATE(1, 16, 1)
FG_NORM_ROTATE(1, 32, 1)
FG_NORM_ROTATE(1, 64, 1)
FG_NORM_ROTATE(1, 64, 2)
FG_NORM_ROTATE(1, 64, 4)

// dw from the workgroups' sums: 16 columns a workgroup, 64 slices of them.
extern "C" __global__ void __launch_bounds__(1024)
    fg_norm_rotate_weight(float* dx, const float* x, const float* w, const int* positions, const float* g, float* dw,
                          const float* partial, int blocks, int tokens, int heads, int dim, int heads_per, float eps,
                          float log2_base_hi, float log2_base_lo) {
  __shared__ float sums[64][16];
  const int col = threadIdx.x % 16, slice = threadIdx.x / 16, d = blockIdx.x * 16 + col;
  float t = 0.f;
  if (d < dim) {
#pragma unroll 4
    for (int b = slice; b < blocks; b += 64) t += partial[static_cast<size_t>(b) * dim + d];
  }
  sums[slice][col] = t;
  __syncthreads();
  // Four runs of 16 slices, then their sum.
  if (slice < 4) {
    t = 0.f;
    for (int k = 0; k < 16; k++) t += sums[16 * slice + k][col];
  }
  __syncthreads();
  if (slice < 4) sums[slice][col] = t;
  __syncthreads();
  if (slice == 0 && d < dim) dw[d] = (sums[0][col] + sums[1][col]) + (sums[2][col] + sums[3][col]);
}
