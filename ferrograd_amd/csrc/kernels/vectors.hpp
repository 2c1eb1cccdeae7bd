// Vectors of floats that start on any float, in rows of any width.
#pragma once

#include <hip/hip_runtime.h>

namespace {

template <int VEC>
struct Unaligned {
  typedef float type __attribute__((ext_vector_type(VEC), aligned(4)));
};
template <>
struct Unaligned<1> {
  typedef float type;
};

template <int VEC>
struct Vec {
  float v[VEC];
};

// `Stream`: past the caches, for what is read once and outputs that would not
// stay in the Infinity Cache.
template <int VEC, bool Stream = false>
__device__ inline Vec<VEC> load(const float* p) {
  typedef typename Unaligned<VEC>::type vec;
  const vec v = Stream ? __builtin_nontemporal_load(reinterpret_cast<const vec*>(p)) : *reinterpret_cast<const vec*>(p);
  Vec<VEC> r;
  if constexpr (VEC == 1) {
    r.v[0] = v;
  } else {
#pragma unroll
    for (int e = 0; e < VEC; e++) r.v[e] = v[e];
  }
  return r;
}

template <int VEC, bool Stream = false>
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

}  // namespace
