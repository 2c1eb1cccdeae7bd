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

}  // namespace

extern "C" __global__ void __launch_bounds__(256)
    fg_dropout(float* __restrict__ out, const float* __restrict__ x, unsigned seed_lo, unsigned seed_hi,
               unsigned offset_lo, unsigned offset_hi, unsigned n_lo, unsigned n_hi, unsigned threshold, float scale) {
  const unsigned long long n = static_cast<unsigned long long>(n_hi) << 32 | n_lo;
  const unsigned long long block = static_cast<unsigned long long>(blockIdx.x) * 256 + threadIdx.x;
  const unsigned long long e = block * 4;
  if (e >= n) return;
  const Words r = philox(static_cast<unsigned>(block), static_cast<unsigned>(block >> 32), offset_lo, offset_hi,
                         seed_lo, seed_hi);
  if (e + 4 <= n) {
    float4 v = *reinterpret_cast<const float4*>(x + e);
    v.x = r.w[0] >= threshold ? v.x * scale : 0.f;
    v.y = r.w[1] >= threshold ? v.y * scale : 0.f;
    v.z = r.w[2] >= threshold ? v.z * scale : 0.f;
    v.w = r.w[3] >= threshold ? v.w * scale : 0.f;
    *reinterpret_cast<float4*>(out + e) = v;
    return;
  }
  for (int i = 0; i < static_cast<int>(n - e); i++) out[e + i] = r.w[i] >= threshold ? x[e + i] * scale : 0.f;
}
