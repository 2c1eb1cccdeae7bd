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
// a workgroup makes the cosines of a few tokens once, in LDS, for all of their
// heads, then goes through their rows in order, a stretch of memory at a time.
// Rows need not start on a vector's alignment, nor halves be whole vectors: the
// last lane of a half then begins where its vector ends with the half, and
// leaves what it shares with the lane before it out of the sums (its stores are
// the same values again). With vectors as wide as the alignment allowed instead,
// 5001 x 7 x 74 took 11 us forward and 16 backward, now 8 and 9.
//
// 16384 tokens of 32 heads of 128: 94 us forward (5.7 TB/s), 140 backward (5.8);
// elementwise kernels reach 6.3 here. Walking rows token by token in waves of
// their own, with angles made per row, backward took 167.
// Angles are formed in 64 bits as revolutions and reduced there: a far position
// times a frequency has more whole turns than 32 bits can hold beside the
// fraction.
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

// A vector of a row, which starts on any float.
template <int VEC>
struct Unaligned {
  typedef float type __attribute__((ext_vector_type(VEC), aligned(4)));
};
template <>
struct Unaligned<1> {
  typedef float type;
};
template <int VEC>
__device__ inline float element(const typename Unaligned<VEC>::type& v, int e) {
  if constexpr (VEC == 1) return v;
  else return v[e];
}

// `Stream`: past the caches, for what is read once and outputs that would not
// stay in the Infinity Cache.
template <int VEC, bool Stream = false>
__device__ inline Vec<VEC> load(const float* p) {
  typedef typename Unaligned<VEC>::type vec;
  const vec v = Stream ? __builtin_nontemporal_load(reinterpret_cast<const vec*>(p)) : *reinterpret_cast<const vec*>(p);
  Vec<VEC> r;
#pragma unroll
  for (int e = 0; e < VEC; e++) r.v[e] = element<VEC>(v, e);
  return r;
}

template <int VEC, bool Stream>
__device__ inline void store(float* p, const Vec<VEC>& r) {
  typedef typename Unaligned<VEC>::type vec;
  vec v;
  if constexpr (VEC == 1) {
    v = r.v[0];
  } else {
#pragma unroll
    for (int e = 0; e < VEC; e++) v[e] = r.v[e];
  }
  if (Stream) __builtin_nontemporal_store(v, reinterpret_cast<vec*>(p));
  else *reinterpret_cast<vec*>(p) = v;
}

template <int G>
__device__ inline float group_sum(float x) {
#pragma unroll
  for (int d = G / 2; d > 0; d /= 2) x += __shfl_xor(x, d, G);
  return x;
}

constexpr int kAngles = 1024;  // of a workgroup's tokens, at most
constexpr int kMaxHalf = 256;

struct Angles {
  double freq[kMaxHalf];  // revolutions per position
  float2 turn[kAngles];   // cos, sin of [token][pair]
};

__device__ inline void frequencies(Angles& a, int half, double log2_base) {
  for (int i = threadIdx.x; i < half; i += kThreads)
    a.freq[i] = exp2(-(static_cast<double>(i) / half) * log2_base) * 0.15915494309189533577;  // 1 / (2 pi)
  __syncthreads();
}

// The angles of `count` tokens; the whole turns go in 64 bits.
__device__ inline void turns(Angles& a, const int* positions, int count, int half) {
  __syncthreads();  // the last tokens' are read
  for (int n = threadIdx.x; n < count * half; n += kThreads) {
    const double t = a.freq[n % half] * positions[n / half];
    sincospif(2.f * static_cast<float>(t - rint(t)), &a.turn[n].y, &a.turn[n].x);
  }
  __syncthreads();
}

// Rows are taken kRows at a time, loaded before the first is worked on: a row is
// a few hundred bytes, and the memory needs more of them under way than there
// are waves. Forward the first are on their way while the angles are made;
// backward that holds too many registers (149 us instead of 143).
constexpr int kRows = 2, kGradRows = 2;

// A lane's part of a row: where its vectors start in the halves, whether it has
// any, and which of their elements are its own.
template <int VEC, int G>
struct Part {
  int at;
  bool any, own[VEC];
  __device__ Part(int half) {
    const int i = static_cast<int>(threadIdx.x) % G * VEC;
    at = min(i, half - VEC);
    any = i < half;
#pragma unroll
    for (int e = 0; e < VEC; e++) own[e] = any && at + e >= i;
  }
};

template <int VEC, int G, bool Stream>
__device__ inline void forward(float* __restrict__ out, const float* __restrict__ x, const float* __restrict__ w,
                               const int* __restrict__ positions, int tokens, int heads, int dim, int per, float eps,
                               float log2_base_hi, float log2_base_lo) {
  __shared__ Angles angles;
  const int half = dim / 2, group = threadIdx.x / G;
  const Part<VEC, G> part(half);
  constexpr int kGroups = kThreads / G;
  const Vec<VEC> wa = load<VEC>(w + part.at), wb = load<VEC>(w + half + part.at);
  bool started = false;
  for (unsigned first = blockIdx.x * per; first < static_cast<unsigned>(tokens); first += gridDim.x * per) {
    const int count = min(per, static_cast<int>(tokens - first)), rows = count * heads;
    const size_t base = static_cast<size_t>(first) * heads * dim + part.at;
    Vec<VEC> a[kRows], b[kRows];
    auto load_rows = [&](int r0) {
#pragma unroll
      for (int k = 0; k < kRows; k++) {
        const float* row = x + base + static_cast<size_t>(min(r0 + k * kGroups, rows - 1)) * dim;
        a[k] = load<VEC, Stream>(row);
        b[k] = load<VEC, Stream>(row + half);
      }
    };
    load_rows(group);  // on their way while the angles are made
    if (!started) frequencies(angles, half, static_cast<double>(log2_base_hi) + log2_base_lo);
    started = true;
    turns(angles, positions + first, count, half);
    for (int r0 = group; r0 < rows; r0 += kRows * kGroups) {
      if (r0 != group) load_rows(r0);
#pragma unroll
      for (int k = 0; k < kRows; k++) {
        const int r = r0 + k * kGroups;
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const float t = a[k].v[e] * a[k].v[e] + b[k].v[e] * b[k].v[e];
          ss += part.own[e] ? t : 0.f;
        }
        const float inv = 1.f / sqrtf(group_sum<G>(ss) / dim + eps);
        if (r >= rows || !part.any) continue;
        const float2* turn = angles.turn + r / heads * half + part.at;
        float* row = out + base + static_cast<size_t>(r) * dim;
        Vec<VEC> ya, yb;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const float2 cs = turn[e];
          const float za = a[k].v[e] * inv * wa.v[e], zb = b[k].v[e] * inv * wb.v[e];
          ya.v[e] = za * cs.x - zb * cs.y;
          yb.v[e] = zb * cs.x + za * cs.y;
        }
        store<VEC, Stream>(row, ya);
        store<VEC, Stream>(row + half, yb);
      }
    }
  }
}

template <int VEC, int G, bool Stream>
__device__ inline void backward(float* __restrict__ dx, const float* __restrict__ x, const float* __restrict__ w,
                                const int* __restrict__ positions, const float* __restrict__ g,
                                float* __restrict__ partial, int tokens, int heads, int dim, int per, float eps,
                                float log2_base_hi, float log2_base_lo) {
  __shared__ Angles angles;
  __shared__ float sums[kThreads * 2 * VEC];  // [group of the workgroup][half][index], index < G * VEC
  const int half = dim / 2, group = threadIdx.x / G;
  const Part<VEC, G> part(half);
  constexpr int kGroups = kThreads / G;
  const Vec<VEC> wa = load<VEC>(w + part.at), wb = load<VEC>(w + half + part.at);
  float da[VEC] = {}, db[VEC] = {};
  frequencies(angles, half, static_cast<double>(log2_base_hi) + log2_base_lo);
  for (unsigned first = blockIdx.x * per; first < static_cast<unsigned>(tokens); first += gridDim.x * per) {
    const int count = min(per, static_cast<int>(tokens - first)), rows = count * heads;
    const size_t base = static_cast<size_t>(first) * heads * dim + part.at;
    Vec<VEC> a[kGradRows], b[kGradRows], p[kGradRows], q[kGradRows];  // x and g
    auto load_rows = [&](int r0) {
#pragma unroll
      for (int k = 0; k < kGradRows; k++) {
        const size_t row = base + static_cast<size_t>(min(r0 + k * kGroups, rows - 1)) * dim;
        a[k] = load<VEC, Stream>(x + row);
        b[k] = load<VEC, Stream>(x + row + half);
        p[k] = load<VEC, Stream>(g + row);
        q[k] = load<VEC, Stream>(g + row + half);
      }
    };
    turns(angles, positions + first, count, half);
    for (int r0 = group; r0 < rows; r0 += kGradRows * kGroups) {
      load_rows(r0);
#pragma unroll
      for (int k = 0; k < kGradRows; k++) {
        const int r = r0 + k * kGroups;
        const float2* turn = angles.turn + min(r, rows - 1) / heads * half + part.at;
        float ss = 0.f, sg = 0.f;  // sums of x^2 and of g' w x
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const float2 cs = turn[e];
          const float ga = p[k].v[e] * cs.x + q[k].v[e] * cs.y;
          const float gb = q[k].v[e] * cs.x - p[k].v[e] * cs.y;
          p[k].v[e] = ga;
          q[k].v[e] = gb;
          const float t = a[k].v[e] * a[k].v[e] + b[k].v[e] * b[k].v[e];
          const float u = ga * wa.v[e] * a[k].v[e] + gb * wb.v[e] * b[k].v[e];
          ss += part.own[e] ? t : 0.f;
          sg += part.own[e] ? u : 0.f;
        }
        const float inv = 1.f / sqrtf(group_sum<G>(ss) / dim + eps);
        const float mean = group_sum<G>(sg) * inv / dim;
        if (r >= rows || !part.any) continue;
        float* row = dx + base + static_cast<size_t>(r) * dim;
        Vec<VEC> oa, ob;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const float na = a[k].v[e] * inv, nb = b[k].v[e] * inv;
          oa.v[e] = inv * (p[k].v[e] * wa.v[e] - na * mean);
          ob.v[e] = inv * (q[k].v[e] * wb.v[e] - nb * mean);
          da[e] += p[k].v[e] * na;
          db[e] += q[k].v[e] * nb;
        }
        store<VEC, Stream>(row, oa);
        store<VEC, Stream>(row + half, ob);
      }
    }
  }
  constexpr int kHalf = G * VEC;
#pragma unroll
  for (int e = 0; e < VEC; e++)
    if (part.own[e]) {
      sums[group * 2 * kHalf + part.at + e] = da[e];
      sums[group * 2 * kHalf + kHalf + part.at + e] = db[e];
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

#define FG_NORM_ROTATE_AS(VEC, G, NAME, STREAM)                                                                     \
  extern "C" __global__ void __launch_bounds__(kThreads) fg_norm_rotate_##NAME(                                     \
      float* out, const float* x, const float* w, const int* positions, int tokens, int heads, int dim, int per,    \
      float eps, float log2_base_hi, float log2_base_lo) {                                                          \
    forward<VEC, G, STREAM>(out, x, w, positions, tokens, heads, dim, per, eps, log2_base_hi, log2_base_lo);        \
  }                                                                                                                 \
  extern "C" __global__ void __launch_bounds__(kThreads) fg_norm_rotate_grad_##NAME(                                \
      float* dx, const float* x, const float* w, const int* positions, const float* g, float* dw, float* partial,   \
      int blocks, int tokens, int heads, int dim, int per, float eps, float log2_base_hi, float log2_base_lo) {     \
    backward<VEC, G, STREAM>(dx, x, w, positions, g, partial, tokens, heads, dim, per, eps, log2_base_hi,           \
                             log2_base_lo);                                                                         \
  }
#define FG_NORM_ROTATE(VEC, G)                       \
  FG_NORM_ROTATE_AS(VEC, G, VEC##_##G, false)        \
  FG_NORM_ROTATE_AS(VEC, G, VEC##_##G##_stream, true)

FG_NORM_ROTATE(1, 8)
FG_NORM_ROTATE(4, 8)
FG_NORM_ROTATE(4, 16)
FG_NORM_ROTATE(4, 32)
FG_NORM_ROTATE(4, 64)

// dw from the workgroups' sums: 16 columns a workgroup, 64 slices of them.
extern "C" __global__ void __launch_bounds__(1024)
    fg_norm_rotate_weight(float* dx, const float* x, const float* w, const int* positions, const float* g, float* dw,
                          const float* partial, int blocks, int tokens, int heads, int dim, int per, float eps,
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
