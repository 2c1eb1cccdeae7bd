// Rows of any width in the registers of L lanes, K vectors of four floats each: L
// a part of a wave, or a workgroup.
#pragma once

#include "vectors.hpp"

namespace {

// The threads of a workgroup that has rows on L lanes each.
constexpr int threads_of(int L) { return L > 256 ? L : 256; }

struct Sum {
  __device__ float operator()(float a, float b) const { return a + b; }
};
struct Largest {  // of the numbers: a NaN is left out
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

// s[0, N) joined over a row's L lanes, in each of them.
template <int L, int N, class Join>
__device__ inline void join_row(float (&s)[N], Join join) {
#pragma unroll
  for (int d = (L < 64 ? L : 64) / 2; d > 0; d /= 2)
#pragma unroll
    for (int n = 0; n < N; n++) s[n] = join(s[n], __shfl_xor(s[n], d));
  if constexpr (L > 64) {
    constexpr int kWaves = L / 64;
    __shared__ float part[kWaves][N];
    __syncthreads();  // the last ones are read
    if (threadIdx.x % 64 == 0)
#pragma unroll
      for (int n = 0; n < N; n++) part[threadIdx.x / 64][n] = s[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; n++) {
      s[n] = part[0][n];
#pragma unroll
      for (int w = 1; w < kWaves; w++) s[n] = join(s[n], part[w][n]);
    }
  }
}

template <int L, int N>
__device__ inline void row_sums(float (&s)[N]) {
  join_row<L>(s, Sum());
}

// A row's columns on a lane: vector k is of the columns from at(k) on. With
// `Whole` rows are of whole vectors, else the last one may end within, and the
// first one begin before the row: `from` is 0, or less.
template <int L, int K, bool Whole>
struct Columns {
  int lane, dim, from = 0;
  __device__ explicit Columns(int d) : lane(static_cast<int>(threadIdx.x) % L), dim(d) {}
  __device__ int at(int k) const { return (k * L + lane) * 4 + (Whole ? 0 : from); }
  __device__ bool whole(int k) const { return Whole ? at(k) < dim : at(k) >= 0 && at(k) + 4 <= dim; }
  // The row, and `past` behind its end.
  template <bool Stream>
  __device__ void read(Vec<4> (&v)[K], const float* row, float past) const {
#pragma unroll
    for (int k = 0; k < K; k++) {
#pragma unroll
      for (int e = 0; e < 4; e++) v[k].v[e] = past;
      if (whole(k)) {
        v[k] = load<4, Stream>(row + at(k));
      } else if (!Whole) {
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (at(k) + e >= 0 && at(k) + e < dim) v[k].v[e] = row[at(k) + e];
      }
    }
  }
  template <bool Stream>
  __device__ void write(float* row, int k, const Vec<4>& v) const {
    if (whole(k)) {
      store<4, Stream>(row + at(k), v);
    } else if (!Whole) {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (at(k) + e >= 0 && at(k) + e < dim) row[at(k) + e] = v.v[e];
    }
  }
};

}  // namespace
