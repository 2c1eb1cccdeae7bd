// Layer norm and its gradients.
//
// Of a row x of D numbers, with m = mean(x), r = (mean((x - m)^2) + eps)^(-1/2):
//   h = (x - m) r,  y = h w + b
// and backward, with u = g w:
//   dx = r (u - mean(u) - h mean(u h)),  dw = sum over rows of g h,  db = sum of g.
//
// Bound by memory: forward reads and writes a row once (8 bytes an element),
// backward reads x and g and writes dx (12). So a row lives in the registers of L
// lanes, K vectors of four each: the mean is taken before the squares of what is
// left (sums of x^2 would lose the digits that a large mean takes), without a
// second read. L is a part of a wave for short rows, a workgroup for long ones.
// dw and db are summed in registers over all rows that a lane sees, then over the
// workgroup, then over the workgroups by a second launch: a fixed order, no
// atomics, and in float32: a lane's rows are all rows over those that the
// workgroups have at a time (from 32768 of 32 columns to 256 of 16384). Registers
// do not hold these sums of more than 16384 columns: x and g are then read again
// for them, in up to 32 parts of the rows. Rows of more than 32768 columns are read
// again for each of their sums.
//
// Rows on 1024 lanes leave a little in scratch memory: 24 bytes a lane backward in
// 4 vectors, 8 in 8, and 36 to 72 forward in 8, where row, weight and bias are 96
// registers of 128.
//
// TB/s of what each must read and write. 16384 rows of 4096: forward 98 us (5.5),
// backward 126 (6.4; 6.6 of all that goes past the L2 caches); of 4095, whose
// vectors are unaligned, 102 and 136. 65536 of 1024: 92 and 120 (5.8 and 6.7); of
// 1023, 101 and 132. 3000 of 20000: 138 (199 with weight and bias read for each
// row), and backward 133 + 90, where reading each row for each sum took 186, and
// 392 + 98.
#include <hip/hip_runtime.h>

#include "rows.hpp"

namespace {

// A row's columns on a lane: its vector k is of those from at(k) on. With `Whole`
// rows are of whole vectors; else the one over the row's end is moved into the
// row, where it shares columns with the lane's before it: sums leave out what a
// lane does not own, and what it does not own it writes as the same value again.
// So each vector is one load and one store (with the last one's elements one by
// one, for which the wave waits, 16384 rows of 4095 took 150 us backward, not 136,
// 131072 of 33 18.4, not 16.1, but 4096 of 16383, which lacks the registers for
// what is moved, 189, not 195: 3% that a second form of the two widest splits
// would save). Rows of less than a vector have no other way.
template <int L, int K, bool Whole>
struct Moved {
  int lane, dim;
  __device__ explicit Moved(int d) : lane(static_cast<int>(threadIdx.x) % L), dim(d) {}
  __device__ int nominal(int k) const { return (k * L + lane) * 4; }
  __device__ bool any(int k) const { return nominal(k) < dim; }
  __device__ int at(int k) const { return Whole ? nominal(k) : max(0, min(nominal(k), dim - 4)); }
  __device__ bool owns(int k, int e) const { return any(k) && (Whole || (at(k) + e >= nominal(k) && at(k) + e < dim)); }
  __device__ bool few() const { return !Whole && L == 8 && dim < 4; }
  // The row's vectors, 0 where there is no column.
  template <bool Stream>
  __device__ void read(Vec<4> (&v)[K], const float* row) const {
#pragma unroll
    for (int k = 0; k < K; k++) {
      v[k] = Vec<4>{};
      if (few()) {
#pragma unroll
        for (int e = 0; e < 3; e++)
          if (owns(k, e)) v[k].v[e] = row[e];
      } else if (any(k)) {
        v[k] = load<4, Stream>(row + at(k));
      }
    }
  }
  template <bool Stream>
  __device__ void write(float* row, int k, const Vec<4>& v) const {
    if (few()) {
#pragma unroll
      for (int e = 0; e < 3; e++)
        if (owns(k, e)) row[e] = v.v[e];
    } else if (any(k)) {
      store<4, Stream>(row + at(k), v);
    }
  }
};

// The row less its mean, and the inverse of its deviation. What a lane has of no
// column is 0 where rows are of whole vectors; else sums leave it out.
struct Moments {
  float mean, inv;
};
template <int L, int K, bool Whole>
__device__ inline Moments centre(Vec<4> (&x)[K], const Moved<L, K, Whole>& cols, float eps) {
  float s[1] = {};
#pragma unroll
  for (int k = 0; k < K; k++)
#pragma unroll
    for (int e = 0; e < 4; e++) s[0] += Whole || cols.owns(k, e) ? x[k].v[e] : 0.f;
  row_sums<L>(s);
  const float mean = s[0] / cols.dim;
  s[0] = 0.f;
#pragma unroll
  for (int k = 0; k < K; k++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      x[k].v[e] = !Whole || cols.any(k) ? x[k].v[e] - mean : 0.f;
      s[0] += Whole || cols.owns(k, e) ? x[k].v[e] * x[k].v[e] : 0.f;
    }
  row_sums<L>(s);
  return {mean, 1.f / sqrtf(s[0] / cols.dim + eps)};
}

template <int L, int K, bool Whole, bool Stream>
__device__ inline void forward(float* __restrict__ out, const float* __restrict__ x, const float* __restrict__ w,
                               const float* __restrict__ b, int rows, int dim, float eps) {
  constexpr int kGroups = threads_of(L) / L;
  const Moved<L, K, Whole> cols(dim);
  Vec<4> vw[K], vb[K] = {};
  cols.template read<false>(vw, w);
  if (b) cols.template read<false>(vb, b);
  for (int r0 = blockIdx.x * kGroups; r0 < rows; r0 += gridDim.x * kGroups) {
    const int r = r0 + static_cast<int>(threadIdx.x) / L;
    Vec<4> v[K];
    cols.template read<false>(v, x + static_cast<size_t>(min(r, rows - 1)) * dim);
    const float inv = centre<L, K, Whole>(v, cols, eps).inv;
    if (r >= rows) continue;
#pragma unroll
    for (int k = 0; k < K; k++) {
#pragma unroll
      for (int e = 0; e < 4; e++) v[k].v[e] = v[k].v[e] * inv * vw[k].v[e] + vb[k].v[e];
      cols.template write<Stream>(out + static_cast<size_t>(r) * dim, k, v[k]);
    }
  }
}

// A workgroup's sums for dw and db go to partial[workgroup][2][dim]. Rows of more
// than one workgroup's 256 lanes keep the weight in LDS: in registers as well it
// would leave room for half the waves. Where K is 8 there is room for no sums: the
// rows' means and deviations go to `stats` for a launch that makes them.
template <int L, int K, bool Whole, bool Stream>
__device__ inline void backward(float* __restrict__ dx, const float* __restrict__ x, const float* __restrict__ w,
                                const float* __restrict__ g, float* __restrict__ partial, float* __restrict__ stats, int rows,
                                int dim, float eps) {
  constexpr bool kSums = K < 8;
  constexpr int kGroups = threads_of(L) / L;
  constexpr bool kHeld = L <= 256;
  __shared__ Vec<4> weights[kHeld ? 1 : K * L];
  const Moved<L, K, Whole> cols(dim);
  Vec<4> vw[K], dw[K] = {}, db[K] = {};
  cols.template read<false>(vw, w);
  if (!kHeld)  // a lane reads back what it wrote
#pragma unroll
    for (int k = 0; k < K; k++) weights[k * L + cols.lane] = vw[k];
  for (int r0 = blockIdx.x * kGroups; r0 < rows; r0 += gridDim.x * kGroups) {
    const int r = r0 + static_cast<int>(threadIdx.x) / L;
    const size_t at = static_cast<size_t>(min(r, rows - 1)) * dim;
    Vec<4> h[K], u[K];
    cols.template read<Stream>(h, x + at);
    cols.template read<Stream>(u, g + at);
    const Moments m = centre<L, K, Whole>(h, cols, eps);
    const float inv = m.inv;
    if (!kSums && threadIdx.x == 0) {
      stats[2 * static_cast<size_t>(r)] = m.mean;
      stats[2 * static_cast<size_t>(r) + 1] = m.inv;
    }
    float s[2] = {};
#pragma unroll
    for (int k = 0; k < K; k++) {
      const Vec<4> wk = kHeld ? vw[k] : weights[k * L + cols.lane];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        // A group past the last row has that row again, and adds none of it.
        const float own = kGroups == 1 || r < rows ? u[k].v[e] : 0.f;
        h[k].v[e] *= inv;
        if (kSums) dw[k].v[e] += own * h[k].v[e];
        if (kSums) db[k].v[e] += own;
        u[k].v[e] *= wk.v[e];
        s[0] += Whole || cols.owns(k, e) ? u[k].v[e] : 0.f;
        s[1] += Whole || cols.owns(k, e) ? u[k].v[e] * h[k].v[e] : 0.f;
      }
    }
    row_sums<L>(s);
    if (r >= rows) continue;
    const float mean = s[0] / dim, slope = s[1] / dim;
#pragma unroll
    for (int k = 0; k < K; k++) {
      Vec<4> d;
#pragma unroll
      for (int e = 0; e < 4; e++) d.v[e] = inv * (u[k].v[e] - mean - h[k].v[e] * slope);
      cols.template write<Stream>(dx + at, k, d);
    }
  }
  if (!kSums) return;
  float* to = partial + static_cast<size_t>(blockIdx.x) * 2 * dim;
  if constexpr (kGroups == 1) {
#pragma unroll
    for (int k = 0; k < K; k++) {
      cols.template write<false>(to, k, dw[k]);
      cols.template write<false>(to + dim, k, db[k]);
    }
  } else {
    __shared__ float sums[kGroups][2][4 * L * K];
    const int group = threadIdx.x / L;
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (cols.any(k)) {
          sums[group][0][cols.at(k) + e] = dw[k].v[e];
          sums[group][1][cols.at(k) + e] = db[k].v[e];
        }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * dim; c += threads_of(L)) {
      float t = 0.f;
#pragma unroll 4
      for (int k = 0; k < kGroups; k++) t += c < dim ? sums[k][0][c] : sums[k][1][c - dim];
      to[c] = t;
    }
  }
}

// ── rows that are read again for each sum ───────────────────────────────────

constexpr int kLong = 1024;  // threads

__device__ inline Moments moments(const float* x, int dim, float eps) {
  float s[1] = {};
  for (int c = threadIdx.x; c < dim; c += kLong) s[0] += x[c];
  row_sums<kLong>(s);
  const float mean = s[0] / dim;
  s[0] = 0.f;
  for (int c = threadIdx.x; c < dim; c += kLong) s[0] += (x[c] - mean) * (x[c] - mean);
  row_sums<kLong>(s);
  return {mean, 1.f / sqrtf(s[0] / dim + eps)};
}

}  // namespace

#define FG_FORWARD_ARGS float *out, const float *x, const float *w, const float *b, int rows, int dim, float eps
// `partial`: [blocks][2][dim]; `stats`: [rows][mean, inverse deviation], of long rows.
#define FG_BACKWARD_ARGS                                                                                              \
  float *dx, const float *x, const float *w, const float *g, float *dw, float *db, float *partial, float *stats, int blocks, \
      int rows, int dim, float eps

#define FG_LAYER_NORM_AS(L, K, NAME, WHOLE, STREAM)                                                                   \
  extern "C" __global__ void __launch_bounds__(threads_of(L)) fg_layer_norm_##NAME(FG_FORWARD_ARGS) {                 \
    forward<L, K, WHOLE, STREAM>(out, x, w, b, rows, dim, eps);                                                       \
  }                                                                                                                   \
  extern "C" __global__ void __launch_bounds__(threads_of(L)) __attribute__((amdgpu_waves_per_eu(4)))                 \
      fg_layer_norm_grad_##NAME(FG_BACKWARD_ARGS) {                                                                   \
    backward<L, K, WHOLE, STREAM>(dx, x, w, g, partial, stats, rows, dim, eps);                                              \
  }
#define FG_LAYER_NORM(L, K)                                  \
  FG_LAYER_NORM_AS(L, K, L##_##K, true, false)               \
  FG_LAYER_NORM_AS(L, K, L##_##K##_stream, true, true)       \
  FG_LAYER_NORM_AS(L, K, L##_##K##_odd, false, false)        \
  FG_LAYER_NORM_AS(L, K, L##_##K##_odd_stream, false, true)

FG_LAYER_NORM(8, 1)
FG_LAYER_NORM(16, 1)
FG_LAYER_NORM(32, 1)
FG_LAYER_NORM(64, 1)
FG_LAYER_NORM(64, 2)
FG_LAYER_NORM(64, 4)
FG_LAYER_NORM(256, 2)
FG_LAYER_NORM(256, 4)
FG_LAYER_NORM(512, 4)
FG_LAYER_NORM(1024, 4)
FG_LAYER_NORM(1024, 8)

extern "C" __global__ void __launch_bounds__(kLong) fg_layer_norm_long(FG_FORWARD_ARGS) {
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const float* row = x + static_cast<size_t>(r) * dim;
    const Moments m = moments(row, dim, eps);
    for (int c = threadIdx.x; c < dim; c += kLong)
      out[static_cast<size_t>(r) * dim + c] = (row[c] - m.mean) * m.inv * w[c] + (b ? b[c] : 0.f);
  }
}

extern "C" __global__ void __launch_bounds__(kLong) fg_layer_norm_grad_long(FG_BACKWARD_ARGS) {
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const size_t at = static_cast<size_t>(r) * dim;
    const Moments m = moments(x + at, dim, eps);
    float s[2] = {};
    for (int c = threadIdx.x; c < dim; c += kLong) {
      const float u = g[at + c] * w[c];
      s[0] += u;
      s[1] += u * ((x[at + c] - m.mean) * m.inv);
    }
    row_sums<kLong>(s);
    const float mean = s[0] / dim, slope = s[1] / dim;
    for (int c = threadIdx.x; c < dim; c += kLong)
      dx[at + c] = m.inv * (g[at + c] * w[c] - mean - (x[at + c] - m.mean) * m.inv * slope);
    if (threadIdx.x == 0) {
      stats[2 * static_cast<size_t>(r)] = m.mean;
      stats[2 * static_cast<size_t>(r) + 1] = m.inv;
    }
  }
}

// A thread sums a column over its part of the rows.
extern "C" __global__ void __launch_bounds__(256) fg_layer_norm_grad_long_sums(FG_BACKWARD_ARGS) {
  const int tiles = (dim + 255) / 256, part = static_cast<int>(blockIdx.x) / tiles;
  const int c = static_cast<int>(blockIdx.x) % tiles * 256 + static_cast<int>(threadIdx.x);
  if (c >= dim) return;
  const int per = (rows + blocks - 1) / blocks, end = min(rows, (part + 1) * per);
  float sw = 0.f, sb = 0.f;
#pragma unroll 4
  for (int r = part * per; r < end; r++) {
    const size_t at = static_cast<size_t>(r) * dim + c;
    sw += g[at] * ((x[at] - stats[2 * static_cast<size_t>(r)]) * stats[2 * static_cast<size_t>(r) + 1]);
    sb += g[at];
  }
  partial[static_cast<size_t>(part) * 2 * dim + c] = sw;
  partial[static_cast<size_t>(part) * 2 * dim + dim + c] = sb;
}

// dw and db from the workgroups' sums: 32 columns of both a workgroup, in 32
// slices of them.
extern "C" __global__ void __launch_bounds__(1024) fg_layer_norm_weight(FG_BACKWARD_ARGS) {
  __shared__ float sums[32][33];
  const int col = threadIdx.x % 32, slice = threadIdx.x / 32, c = blockIdx.x * 32 + col;
  float t = 0.f;
  if (c < 2 * dim) {
#pragma unroll 8
    for (int k = slice; k < blocks; k += 32) t += partial[static_cast<size_t>(k) * 2 * dim + c];
  }
  sums[slice][col] = t;
  __syncthreads();
  // A column's slices are on 32 lanes.
  t = sums[col][slice];
#pragma unroll
  for (int d = 16; d > 0; d /= 2) t += __shfl_xor(t, d, 32);
  const int at = blockIdx.x * 32 + slice;
  if (col != 0) return;
  if (at < dim) dw[at] = t;
  else if (at < 2 * dim && db) db[at - dim] = t;
}
