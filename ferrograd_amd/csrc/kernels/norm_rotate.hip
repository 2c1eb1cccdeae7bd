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

// `stream`: past the caches.
template <int VEC>
__device__ inline void store(float* p, const Vec<VEC>& r, bool stream) {
  typedef float vec __attribute__((ext_vector_type(VEC)));
  vec v;
#pragma unroll
  for (int e = 0; e < VEC; e++) v[e] = r.v[e];
  if (stream) __builtin_nontemporal_store(v, reinterpret_cast<vec*>(p));
  else *reinterpret_cast<vec*>(p) = v;
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
// units g, g + groups, ... Heads are taken kHeads at a time, loaded before the
// first is worked on: a row is a few hundred bytes, and the memory needs more
// of them under way than there are waves.
constexpr int kHeads = 4, kGradHeads = 2;

template <int VEC, int G, int NV>
__device__ inline void forward(float* __restrict__ out, const float* __restrict__ x, const float* __restrict__ w,
                               const int* __restrict__ positions, int tokens, int heads, int dim, int heads_per,
                               float eps, float log2_base_hi, float log2_base_lo, bool stream) {
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
    for (int h = h0; h < h1; h += kHeads) {
      Vec<VEC> a[kHeads][NV], b[kHeads][NV];
#pragma unroll
      for (int k = 0; k < kHeads; k++) {
        const float* row = x + (static_cast<size_t>(token) * heads + min(h + k, h1 - 1)) * dim;
#pragma unroll
        for (int v = 0; v < NV; v++) {
          const int i = (v * G + sub) * VEC;
          if (i < half) {
            a[k][v] = load<VEC>(row + i);
            b[k][v] = load<VEC>(row + half + i);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kHeads; k++) {
        float ss = 0.f;
#pragma unroll
        for (int v = 0; v < NV; v++)
          if ((v * G + sub) * VEC < half) {
#pragma unroll
            for (int e = 0; e < VEC; e++) ss += a[k][v].v[e] * a[k][v].v[e] + b[k][v].v[e] * b[k][v].v[e];
          }
        const float r = 1.f / sqrtf(group_sum<G>(ss) / dim + eps);
        if (h + k >= h1) continue;
        float* row = out + (static_cast<size_t>(token) * heads + h + k) * dim;
#pragma unroll
        for (int v = 0; v < NV; v++) {
          const int i = (v * G + sub) * VEC;
          if (i >= half) continue;
          Vec<VEC> ya, yb;
#pragma unroll
          for (int e = 0; e < VEC; e++) {
            const float za = a[k][v].v[e] * r * wa[v].v[e], zb = b[k][v].v[e] * r * wb[v].v[e];
            ya.v[e] = za * c[v][e] - zb * s[v][e];
            yb.v[e] = zb * c[v][e] + za * s[v][e];
          }
          store<VEC>(row + i, ya, stream);
          store<VEC>(row + half + i, yb, stream);
        }
      }
    }
  }
}

template <int VEC, int G, int NV>
__device__ inline void backward(float* __restrict__ dx, const float* __restrict__ x, const float* __restrict__ w,
                                const int* __restrict__ positions, const float* __restrict__ g,
                                float* __restrict__ partial, int tokens, int heads, int dim, int heads_per, float eps,
                                float log2_base_hi, float log2_base_lo, bool stream) {
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
    for (int h = h0; h < h1; h += kGradHeads) {
      Vec<VEC> a[kGradHeads][NV], b[kGradHeads][NV], p[kGradHeads][NV], q[kGradHeads][NV];  // x and g
#pragma unroll
      for (int k = 0; k < kGradHeads; k++) {
        const size_t row = (static_cast<size_t>(token) * heads + min(h + k, h1 - 1)) * dim;
#pragma unroll
        for (int v = 0; v < NV; v++) {
          const int i = (v * G + sub) * VEC;
          if (i < half) {
            a[k][v] = load<VEC>(x + row + i);
            b[k][v] = load<VEC>(x + row + half + i);
            p[k][v] = load<VEC>(g + row + i);
            q[k][v] = load<VEC>(g + row + half + i);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kGradHeads; k++) {
        float ss = 0.f, sg = 0.f;  // sums of x^2 and of g' w x
#pragma unroll
        for (int v = 0; v < NV; v++) {
          if ((v * G + sub) * VEC >= half) continue;
#pragma unroll
          for (int e = 0; e < VEC; e++) {
            const float ga = p[k][v].v[e] * c[v][e] + q[k][v].v[e] * s[v][e];
            const float gb = q[k][v].v[e] * c[v][e] - p[k][v].v[e] * s[v][e];
            p[k][v].v[e] = ga;
            q[k][v].v[e] = gb;
            ss += a[k][v].v[e] * a[k][v].v[e] + b[k][v].v[e] * b[k][v].v[e];
            sg += ga * wa[v].v[e] * a[k][v].v[e] + gb * wb[v].v[e] * b[k][v].v[e];
          }
        }
        const float r = 1.f / sqrtf(group_sum<G>(ss) / dim + eps);
        const float mean = group_sum<G>(sg) * r / dim;
        if (h + k >= h1) continue;
        float* row = dx + (static_cast<size_t>(token) * heads + h + k) * dim;
#pragma unroll
        for (int v = 0; v < NV; v++) {
          const int i = (v * G + sub) * VEC;
          if (i >= half) continue;
          Vec<VEC> oa, ob;
#pragma unroll
          for (int e = 0; e < VEC; e++) {
            const float na = a[k][v].v[e] * r, nb = b[k][v].v[e] * r;
            oa.v[e] = r * (p[k][v].v[e] * wa[v].v[e] - na * mean);
            ob.v[e] = r * (q[k][v].v[e] * wb[v].v[e] - nb * mean);
            da[v][e] += p[k][v].v[e] * na;
            db[v][e] += q[k][v].v[e] * nb;
          }
          store<VEC>(row + i, oa, stream);
          store<VEC>(row + half + i, ob, stream);
        }
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
      float eps, float log2_base_hi, float log2_base_lo, int stream) {                                                 \
    forward<VEC, G, NV>(out, x, w, positions, tokens, heads, dim, heads_per, eps, log2_base_hi, log2_base_lo,          \
                          stream);                                                                                     \
  }                                                                                                                    \
  extern "C" __global__ void __launch_bounds__(kThreads) fg_norm_rotate_grad_##VEC##_##G##_##NV(                       \
      float* dx, const float* x, const float* w, const int* positions, const float* g, float* dw, float* partial,      \
      int blocks, int tokens, int heads, int dim, int heads_per, float eps, float log2_base_hi, float log2_base_lo,    \
      int stream) {                                                                                                    \
    backward<VEC, G, NV>(dx, x, w, positions, g, partial, tokens, heads, dim, heads_per, eps, log2_base_hi,            \
                         log2_base_lo, stream);                                                                        \
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
                          float log2_base_hi, float log2_base_lo, int stream) {
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
