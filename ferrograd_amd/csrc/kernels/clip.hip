// The norm of all elements of many tensors together, and their clipping to it.
//
//   norm = sqrt(sum of x^2),  y = x * max_norm / max(norm, max_norm)
// Squares and sums are in 64 bits: they neither overflow nor vanish, and the
// rate of a double's multiply-add hides behind the memory's. A norm of NaN
// makes every y NaN, one of infinity 0 (NaN where x is infinite).
//
// 151 million numbers: squares 93 us (6.5 TB/s), products 216 (5.6); 136 and 211
// where everything goes through the caches in its order. 67 million: 42 + 83 (6.3
// and 6.5), and 70 + 84.
//
// A launch takes up to 64 tensors, one for each lane of a wave: the lanes hold
// the tensors' addresses and sizes, read out of the launch's arguments, and the
// running count of their chunks, so that a ballot finds a chunk's tensor. More
// tensors go in several launches, each adding to the sums of the one before.
#include <hip/hip_runtime.h>

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;  // elements a workgroup takes at a time
constexpr int kVectors = kChunk / 4 / kThreads;
// The second pass goes through the chunks from the last one on: of many, the
// first pass leaves this many in the Infinity Cache for it, and reads the others
// past it.
constexpr int kKept = 8192;

typedef float floatx4 __attribute__((ext_vector_type(4)));
#define FG_CONSTANT __attribute__((address_space(4)))
#define FG_GLOBAL __attribute__((address_space(1)))

// A lane's tensor, of a launch's TENSORS.
template <int TENSORS>
struct Mine {
  unsigned long long in, out;
  int end;   // chunks of the tensors up to this one
  int last;  // elements of its last chunk

  // The launch's arguments begin with their addresses and sizes, and, where there
  // are `outputs`, those' addresses.
  __device__ Mine(int count, bool outputs) : in(0), out(0) {
    const auto* args = (const FG_CONSTANT unsigned long long*)__builtin_amdgcn_kernarg_segment_ptr();
    const int lane = threadIdx.x % 64;
    unsigned long long n = 0;
    if (lane < count) {
      in = args[lane];
      n = args[TENSORS + lane];
      if (outputs) out = args[2 * TENSORS + lane];
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
  template <int TENSORS>
  __device__ Chunk(const Mine<TENSORS>& t, int c) {
    const int i = __popcll(__ballot(t.end <= c));
    const size_t at = static_cast<size_t>(c - (i ? __builtin_amdgcn_readlane(t.end, i - 1) : 0)) * kChunk;
    in = reinterpret_cast<const FG_GLOBAL float*>(of_lane(t.in, i)) + at;
    out = reinterpret_cast<FG_GLOBAL float*>(of_lane(t.out, i)) + at;
    n = c + 1 == __builtin_amdgcn_readlane(t.end, i) ? __builtin_amdgcn_readlane(t.last, i) : kChunk;
  }
};

// A whole chunk's vectors of a thread; `Past` the caches.
template <bool Past>
__device__ inline void read(floatx4 (&v)[kVectors], const FG_GLOBAL float* in) {
  const FG_GLOBAL floatx4* from = reinterpret_cast<const FG_GLOBAL floatx4*>(in) + threadIdx.x;
#pragma unroll
  for (int i = 0; i < kVectors; i++) v[i] = Past ? __builtin_nontemporal_load(from + i * kThreads) : from[i * kThreads];
}

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

// `Stream`: outputs past the caches, for those that would not stay there.
template <int TENSORS, bool Stream>
__device__ inline void clip(const double* sums, float* total, double max_norm, int blocks, int count) {
  const Mine<TENSORS> t(count, true);
  const int chunks = t.chunks();
  const double norm = norm_of(sums, blocks);
  if (total && blockIdx.x == 0 && threadIdx.x == 0) *total = static_cast<float>(norm);
  // Not fmax, which would take max_norm for a NaN.
  double factor = max_norm / (norm <= max_norm ? max_norm : norm);
  // A factor below float32's normal range would lose its digits, though not all
  // products with it are that small: it goes in two steps, its digits and its
  // power of two.
  int power = 0;
  if (factor < 0x1p-126) factor = frexp(factor, &power);
  const float scale = static_cast<float>(factor);
  power = __builtin_amdgcn_readfirstlane(power);  // the same in all threads
  auto clipped = [&](float x) { return power ? ldexpf(x * scale, power) : x * scale; };
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const Chunk k(t, chunks - 1 - c);
    if (k.n == kChunk) {
      floatx4 v[kVectors];
      read<false>(v, k.in);
      FG_GLOBAL floatx4* to = reinterpret_cast<FG_GLOBAL floatx4*>(k.out) + threadIdx.x;
#pragma unroll
      for (int i = 0; i < kVectors; i++) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[i][e] = clipped(v[i][e]);
        if (Stream) __builtin_nontemporal_store(v[i], to + i * kThreads);
        else to[i * kThreads] = v[i];
      }
    } else {
      for (int i = threadIdx.x; i < k.n; i += kThreads) k.out[i] = clipped(k.in[i]);
    }
  }
}

// A workgroup's squares in its chunks from c on that are below `end`.
template <bool Past, int TENSORS>
__device__ inline double squares(const Mine<TENSORS>& t, int& c, int end) {
  double s = 0.0;
  for (; c < end; c += gridDim.x) {
    const Chunk k(t, c);
    if (k.n == kChunk) {
      floatx4 v[kVectors];
      read<Past>(v, k.in);
#pragma unroll
      for (int i = 0; i < kVectors; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) s += static_cast<double>(v[i][e]) * v[i][e];
    } else {
      for (int i = threadIdx.x; i < k.n; i += kThreads) s += static_cast<double>(k.in[i]) * k.in[i];
    }
  }
  return s;
}

// A workgroup's sum of squares, and what `before` (if any) has in its place.
template <int TENSORS>
__device__ inline void square_sums(double* sums, const double* before, int count) {
  const Mine<TENSORS> t(count, false);
  const int chunks = t.chunks();
  int c = blockIdx.x;
  double s = squares<true>(t, c, chunks - kKept);
  s += squares<false>(t, c, chunks);
  s = block_sum(s);
  if (threadIdx.x == 0) sums[blockIdx.x] = before ? before[blockIdx.x] + s : s;
}

}  // namespace

#define FG_8(T, p) T p##0, T p##1, T p##2, T p##3, T p##4, T p##5, T p##6, T p##7
#define FG_16(T, p) FG_8(T, p##0), FG_8(T, p##1)
#define FG_64(T, p) FG_16(T, p##0), FG_16(T, p##1), FG_16(T, p##2), FG_16(T, p##3)

// Of up to 16 tensors, with fewer arguments to pass, and of up to 64.
#define FG_CLIP_AS(N, NAME, STREAM)                                                                               \
  extern "C" __global__ void __launch_bounds__(kThreads)                                                          \
      fg_clip_##NAME(FG_##N(const float*, in), FG_##N(long long, n), FG_##N(float*, out), const double* sums,     \
                     float* total, double max_norm, int blocks, int count) {                                      \
    clip<N, STREAM>(sums, total, max_norm, blocks, count);                                                        \
  }
#define FG_CLIP(N)                                                                                                \
  extern "C" __global__ void __launch_bounds__(kThreads)                                                          \
      fg_square_sums_##N(FG_##N(const float*, in), FG_##N(long long, n), double* sums, const double* before, int count) { \
    square_sums<N>(sums, before, count);                                                                          \
  }                                                                                                               \
  FG_CLIP_AS(N, N, false)                                                                                         \
  FG_CLIP_AS(N, N##_stream, true)

FG_CLIP(16)
FG_CLIP(64)

extern "C" __global__ void __launch_bounds__(kThreads) fg_norm_of_sums(float* out, const double* sums, int blocks) {
  const double norm = norm_of(sums, blocks);
  if (threadIdx.x == 0) *out = static_cast<float>(norm);
}
