// The norm of all elements of many tensors together, and their clipping to it.
//
//   norm = sqrt(sum of x^2),  y = x * max_norm / max(norm, max_norm)
// Squares and sums are in 64 bits: they neither overflow nor vanish, and the
// rate of a double's multiply-add hides behind the memory's. A norm of NaN
// makes every y NaN, one of infinity 0 (NaN where x is infinite).
//
// A launch takes up to 64 tensors, one for each lane of a wave: the lanes hold
// the tensors' addresses and sizes, read out of the launch's arguments, and the
// running count of their chunks, so that a ballot finds a chunk's tensor. More
// tensors go in several launches, each adding to the sums of the one before.
#include <hip/hip_runtime.h>

namespace {

constexpr int kThreads = 256, kTensors = 64;
constexpr int kChunk = 4096;  // elements a workgroup takes at a time
constexpr int kVectors = kChunk / 4 / kThreads;

typedef float floatx4 __attribute__((ext_vector_type(4)));
#define FG_CONSTANT __attribute__((address_space(4)))
#define FG_GLOBAL __attribute__((address_space(1)))

// A lane's tensor.
struct Mine {
  unsigned long long in, out;
  int end;   // chunks of the tensors up to this one
  int last;  // elements of its last chunk

  // The launch's arguments begin with 64 addresses and 64 sizes, and, where
  // there are `outputs`, 64 addresses of theirs.
  __device__ Mine(int count, bool outputs) : in(0), out(0) {
    const auto* args = (const FG_CONSTANT unsigned long long*)__builtin_amdgcn_kernarg_segment_ptr();
    const int lane = threadIdx.x % 64;
    unsigned long long n = 0;
    if (lane < count) {
      in = args[lane];
      n = args[kTensors + lane];
      if (outputs) out = args[2 * kTensors + lane];
    }
    end = static_cast<int>((n + kChunk - 1) / kChunk);
    last = static_cast<int>((n - 1) % kChunk) + 1;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int before = __shfl_up(end, d);
      if (lane >= d) end += before;
    }
  }
  __device__ int chunks() const { return __builtin_amdgcn_readlane(end, 63); }
};

__device__ inline unsigned long long of_lane(unsigned long long x, int lane) {
  return static_cast<unsigned long long>(static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(x >> 32), lane))) << 32 |
         static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(x), lane));
}

// Chunk c (below chunks()) of the tensors: where it is, and how long. Its length
// is found in 32 bits: a uniform minimum in 64 came out of the compiler (ROCm
// 7.2) as a select on a condition that its comparison had not set.
struct Chunk {
  const FG_GLOBAL float* in;
  FG_GLOBAL float* out;
  int n;
  __device__ Chunk(const Mine& t, int c) {
    const int i = __popcll(__ballot(t.end <= c));
    const size_t at = static_cast<size_t>(c - (i ? __builtin_amdgcn_readlane(t.end, i - 1) : 0)) * kChunk;
    in = reinterpret_cast<const FG_GLOBAL float*>(of_lane(t.in, i)) + at;
    out = reinterpret_cast<FG_GLOBAL float*>(of_lane(t.out, i)) + at;
    n = c + 1 == __builtin_amdgcn_readlane(t.end, i) ? __builtin_amdgcn_readlane(t.last, i) : kChunk;
  }
};

// The sum over a workgroup, in every thread, the same in each launch.
__device__ inline double block_sum(double x) {
  __shared__ double part[kThreads / 64];
#pragma unroll
  for (int d = 32; d > 0; d /= 2) x += __shfl_xor(x, d);
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = x;
  __syncthreads();
  x = 0.0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; i++) x += part[i];
  return x;
}

__device__ inline double norm_of(const double* sums, int blocks) {
  double s = 0.0;
  for (int i = threadIdx.x; i < blocks; i += kThreads) s += sums[i];
  return sqrt(block_sum(s));
}

}  // namespace

#define FG_8(T, p) T p##0, T p##1, T p##2, T p##3, T p##4, T p##5, T p##6, T p##7
#define FG_64(T, p) FG_8(T, p##0), FG_8(T, p##1), FG_8(T, p##2), FG_8(T, p##3), FG_8(T, p##4), FG_8(T, p##5), FG_8(T, p##6), FG_8(T, p##7)

// A workgroup's sum of squares, and what `before` (if any) has in its place.
extern "C" __global__ void __launch_bounds__(kThreads)
    fg_square_sums(FG_64(const float*, in), FG_64(long long, n), double* sums, const double* before, int count) {
  const Mine t(count, false);
  const int chunks = t.chunks();
  double s = 0.0;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const Chunk k(t, c);
    if (k.n == kChunk) {
      floatx4 v[kVectors];
#pragma unroll
      for (int i = 0; i < kVectors; i++) v[i] = reinterpret_cast<const FG_GLOBAL floatx4*>(k.in)[i * kThreads + threadIdx.x];
#pragma unroll
      for (int i = 0; i < kVectors; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) s += static_cast<double>(v[i][e]) * v[i][e];
    } else {
      for (int i = threadIdx.x; i < k.n; i += kThreads) s += static_cast<double>(k.in[i]) * k.in[i];
    }
  }
  s = block_sum(s);
  if (threadIdx.x == 0) sums[blockIdx.x] = before ? before[blockIdx.x] + s : s;
}

extern "C" __global__ void __launch_bounds__(kThreads) fg_norm_of_sums(float* out, const double* sums, int blocks) {
  const double norm = norm_of(sums, blocks);
  if (threadIdx.x == 0) *out = static_cast<float>(norm);
}

extern "C" __global__ void __launch_bounds__(kThreads)
    fg_clip(FG_64(const float*, in), FG_64(long long, n), FG_64(float*, out), const double* sums, float* total,
            double max_norm, int blocks, int count) {
  const Mine t(count, true);
  const int chunks = t.chunks();
  const double norm = norm_of(sums, blocks);
  if (total && blockIdx.x == 0 && threadIdx.x == 0) *total = static_cast<float>(norm);
  // Not fmax, which would take max_norm for a NaN.
  const float scale = static_cast<float>(max_norm / (norm <= max_norm ? max_norm : norm));
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const Chunk k(t, c);
    if (k.n == kChunk) {
      floatx4 v[kVectors];
#pragma unroll
      for (int i = 0; i < kVectors; i++) v[i] = reinterpret_cast<const FG_GLOBAL floatx4*>(k.in)[i * kThreads + threadIdx.x];
#pragma unroll
      for (int i = 0; i < kVectors; i++) reinterpret_cast<FG_GLOBAL floatx4*>(k.out)[i * kThreads + threadIdx.x] = v[i] * scale;
    } else {
      for (int i = threadIdx.x; i < k.n; i += kThreads) k.out[i] = k.in[i] * scale;
    }
  }
}
