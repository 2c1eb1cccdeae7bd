// Dropout from a counter-based generator: nothing about the mask is stored,
// the gradient draws the same words again.
//
// y_e = x_e / (1 - p) where word_e >= floor(p 2^32), else 0. word_e is word
// e % 4 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers:
// as easy as 1, 2, 3", 2011) of the counter (e / 4, offset) under the key
// `seed`, each 64 bits as (low, high) words. A dropped element is 0 whatever
// it held.
#include <hip/hip_runtime.h>

namespace {

struct Words {
  unsigned w[4];
};

__device__ inline Words philox(unsigned c0, unsigned c1, unsigned c2, unsigned c3, unsigned k0, unsigned k1) {
#pragma unroll
  for (int round = 0; round < 10; round++) {
    const unsigned long long x = static_cast<unsigned long long>(c0) * 0xD2511F53u;
    const unsigned long long y = static_cast<unsigned long long>(c2) * 0xCD9E8D57u;
    c0 = static_cast<unsigned>(y >> 32) ^ c1 ^ k0;
    c1 = static_cast<unsigned>(y);
    c2 = static_cast<unsigned>(x >> 32) ^ c3 ^ k1;
    c3 = static_cast<unsigned>(x);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// A thread draws one block of words for four elements; the draws hide behind
// the memory. 131 MB in and out, out of four buffers each in turn: 128 threads
// 42.8 us (6.1 TB/s), with loads and stores past the caches (`Stream`) 39.6
// (6.6); 256 threads 43.4 and 39.9; four blocks a thread 48.0 and 44.1; without
// the generator's rounds 43.2 and 40.2. From the Infinity Cache 32.8, which
// loads past it give up: only outputs too large for it stream.
typedef float floatx4 __attribute__((ext_vector_type(4)));

template <bool Stream>
__device__ inline void dropout(float* __restrict__ out, const float* __restrict__ x, unsigned seed_lo, unsigned seed_hi,
                               unsigned offset_lo, unsigned offset_hi, unsigned n_lo, unsigned n_hi, unsigned threshold,
                               float scale) {
  const unsigned long long n = static_cast<unsigned long long>(n_hi) << 32 | n_lo;
  const unsigned long long block = static_cast<unsigned long long>(blockIdx.x) * 128 + threadIdx.x;
  const unsigned long long e = block * 4;
  if (e >= n) return;
  const Words r = philox(static_cast<unsigned>(block), static_cast<unsigned>(block >> 32), offset_lo, offset_hi,
                         seed_lo, seed_hi);
  if (e + 4 <= n) {
    const floatx4* from = reinterpret_cast<const floatx4*>(x + e);
    floatx4* to = reinterpret_cast<floatx4*>(out + e);
    floatx4 v = Stream ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = r.w[i] >= threshold ? v[i] * scale : 0.f;
    if (Stream) __builtin_nontemporal_store(v, to);
    else *to = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; i++)
    if (e + i < n) out[e + i] = r.w[i] >= threshold ? x[e + i] * scale : 0.f;
}

}  // namespace

extern "C" __global__ void __launch_bounds__(128)
    fg_dropout(float* out, const float* x, unsigned seed_lo, unsigned seed_hi, unsigned offset_lo, unsigned offset_hi,
               unsigned n_lo, unsigned n_hi, unsigned threshold, float scale) {
  dropout<false>(out, x, seed_lo, seed_hi, offset_lo, offset_hi, n_lo, n_hi, threshold, scale);
}

extern "C" __global__ void __launch_bounds__(128)
    fg_dropout_stream(float* out, const float* x, unsigned seed_lo, unsigned seed_hi, unsigned offset_lo,
                      unsigned offset_hi, unsigned n_lo, unsigned n_hi, unsigned threshold, float scale) {
  dropout<true>(out, x, seed_lo, seed_hi, offset_lo, offset_hi, n_lo, n_hi, threshold, scale);
}
