// Attention and its gradients.
//
//   S_ij = scale q_i . k_j over the keys j that query i sees, y_i = softmax(S_i) v
// Query head h of batch b reads key head h / (Hq / Hk). Keys at or past
// lengths[b] are hidden, and with `causal` those past i + Sk - Sq. A query that
// sees no key gives 0 and gradients of 0.
// Matrices are one row per token: q, y [B Sq, Hq D], k, v [B Sk, Hk D].
// stats holds per (b, h, i) m_i, no less than the row's maximum of S log2 e less
// kLazy, then 1 / sum_j exp2(S_ij log2 e - m_i), for the gradients to make the
// probabilities again.
#include <hip/hip_runtime.h>

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

struct Shape {
  int b, sq, sk, hq, hk, d, causal;
};

// Keys of batch b.
__device__ inline int key_count(const Shape& s, const int* lengths, int b) {
  return lengths ? min(max(lengths[b], 0), s.sk) : s.sk;
}

// Keys that query i sees: those below this.
__device__ inline int visible(const Shape& s, int keys, int i) {
  return s.causal ? max(0, min(keys, i + s.sk - s.sq + 1)) : keys;
}

// 1 / a row's sum: 0 where it saw no key, and NaN where one of its scores was, so
// that its gradients are not finite either.
__device__ inline float inverse_sum(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }

// The word joined over eight lanes next to each other, and over a wave, in all
// of them: by lane permutations of the vector unit, none of which passes LDS.
template <class Join>
__device__ inline int join8(int x, Join join) {
  x = join(x, __builtin_amdgcn_mov_dpp(x, 0xB1, 0xF, 0xF, false));   // lanes 1, 0, 3, 2 of four
  x = join(x, __builtin_amdgcn_mov_dpp(x, 0x4E, 0xF, 0xF, false));   // lanes 2, 3, 0, 1 of four
  return join(x, __builtin_amdgcn_mov_dpp(x, 0x141, 0xF, 0xF, false));  // eight mirrored
}
template <class Join>
__device__ inline int join_wave(int x, Join join) {
  x = join8(x, join);
  x = join(x, __builtin_amdgcn_mov_dpp(x, 0x140, 0xF, 0xF, false));  // sixteen mirrored
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = join(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return join(b[0], b[1]);
}
__device__ inline int max_of_floats(int a, int b) { return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b))); }

__device__ inline float sum8(float x) {
  return __int_as_float(join8(__float_as_int(x), [](int a, int b) {
    return __float_as_int(__int_as_float(a) + __int_as_float(b));
  }));
}
__device__ inline float wave_max(float x) { return __int_as_float(join_wave(__float_as_int(x), max_of_floats)); }

// ── products of cut operands ────────────────────────────────────────────────
// A float32 product on the float16 matrix cores: each operand is scaled by a
// power of two that brings its block's largest value below 2^15 and cut into
// two float16 parts, 11 bits each, and a b = a1 b1 + a1 b2 + a2 b1 with sums in
// float32; a2 b2, 2^-21 of the product at most, is left out. Three float16
// products cost less than a fifth of one float32 product's matrix-core time. That
// is 22 bits of each number instead of float32's 24; measured against 64 bits,
// results are off by 5e-7 to 1e-6, which is what float32's own sums of this length are.

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

// Rows of a block that shares a scale, and of a tile.
constexpr int kBlock = 32;
// The exponents of blocks: at most kMostExponent, or, beyond every sum of two of
// these, that of a block of zeros, which takes part in nothing, and that of one
// that is not finite, nor is what it takes part in.
constexpr int kMostExponent = 127, kNoExponent = 500, kNotFiniteExponent = 900, kZeroExponent = 1000;
constexpr int kPart = 1024;  // bytes of one fragment: 64 lanes of 8 float16

// The power of two that brings `top`, a block's largest magnitude, into
// [2^14, 2^15).
__device__ inline int block_exponent(float top) {
  if (top == 0.f) return kZeroExponent;
  if (!(top < INFINITY)) return kNotFiniteExponent;
  int e;
  frexpf(top, &e);  // top = f 2^e with f in [1/2, 1)
  return min(15 - e, kMostExponent);
}

// The scale of a block of exponent e.
__device__ inline float block_scale(int e) { return e < kNoExponent ? ldexpf(1.f, e) : e == kZeroExponent ? 0.f : 1.f; }

// Eight scaled numbers as two parts, both rounded to nearest.
__device__ inline void cut(const float (&x)[8], half8* hi, half8* lo) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const _Float16 h = static_cast<_Float16>(x[i]);
    (*hi)[i] = h;
    (*lo)[i] = static_cast<_Float16>(x[i] - static_cast<float>(h));
  }
}

// The larger of the two halves of a wave, in both.
__device__ inline float halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ inline floatx16 mfma(half8 a, half8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ inline floatx16 mfma3(half8 ah, half8 al, half8 bh, half8 bl, floatx16 c) {
  c = mfma(al, bh, c);
  c = mfma(ah, bl, c);
  return mfma(ah, bh, c);
}

// Fragments. A 32x32x16 product takes of its operands' rows (or columns) n and
// terms k, in lane l, n = l % 32 and k = 8 (l / 32) + 0..7, and gives in lane l
// column l % 32 and rows result_row(r, l / 32), r < 16. Rows that a later
// product sums over are taken in the order in which results hold them:
// registers 8u .. 8u + 7 of the lane are its eight terms of step u.
__device__ inline int result_row(int r, int half) { return 8 * (r / 4) + 4 * half + r % 4; }

// A block of 32 rows as fragments of a product over its columns: for each 16
// columns the first parts, then the second.
template <int NB>
constexpr int kRowBytes = NB * 2 * 2 * kPart;
// ... of a product over its rows: for each 32 columns and each 16 rows (in the
// order of results) the first parts, then the second.
template <int NB>
constexpr int kColBytes = NB * 2 * 2 * kPart;

// A tile ends with a page of numbers of its blocks: read from LDS like the
// rest. (A load of one inside the loop would wait for the copies before it.)
constexpr int kTail = kPart;

// One block, x[row][column] in LDS (rows of kStride floats), times 2^e.
template <int NB>
constexpr int kStride = NB * 32 + 4;

template <int NB>
__device__ inline void write_rows(const float* x, float scale, char* out) {
  for (int g = threadIdx.x; g < NB * 2 * 64; g += 256) {
    const int t = g / 64, lane = g % 64;
    const float* p = x + (lane % 32) * kStride<NB> + 16 * t + 8 * (lane / 32);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = p[i] * scale;
    half8 hi, lo;
    cut(v, &hi, &lo);
    *reinterpret_cast<half8*>(out + t * 2 * kPart + lane * 16) = hi;
    *reinterpret_cast<half8*>(out + t * 2 * kPart + kPart + lane * 16) = lo;
  }
}

template <int NB>
__device__ inline void write_cols(const float* x, float scale, char* out) {
  for (int g = threadIdx.x; g < NB * 2 * 64; g += 256) {
    const int t = g / 64, lane = g % 64;  // t = 2 * (32 columns) + (16 rows)
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
      v[i] = x[result_row(8 * (t % 2) + i, lane / 32) * kStride<NB> + 32 * (t / 2) + lane % 32] * scale;
    half8 hi, lo;
    cut(v, &hi, &lo);
    *reinterpret_cast<half8*>(out + t * 2 * kPart + lane * 16) = hi;
    *reinterpret_cast<half8*>(out + t * 2 * kPart + kPart + lane * 16) = lo;
  }
}

// The largest of the 256 threads' values, in all of them. `shared`: 4 floats.
__device__ inline float block_max(float x, float* shared) {
  x = wave_max(x);
  if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = x;
  __syncthreads();
  x = fmaxf(fmaxf(shared[0], shared[1]), fmaxf(shared[2], shared[3]));
  return x;
}

// A block's largest magnitude (infinite where it holds a NaN) and its smallest
// that is not zero.
struct Extremes {
  float top = 0.f, least = INFINITY;
  __device__ void take(const float4& v) {
    const float a[4] = {fabsf(v.x), fabsf(v.y), fabsf(v.z), fabsf(v.w)};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      top = a[i] == a[i] ? fmaxf(top, a[i]) : INFINITY;
      least = fminf(least, a[i] > 0.f ? a[i] : INFINITY);
    }
  }
  // Those of the 256 threads, in all of them. `shared`: 8 floats.
  __device__ void join(float* shared) {
    const float t = wave_max(top), l = wave_max(-least);
    if (threadIdx.x % 64 == 0) {
      shared[threadIdx.x / 64] = t;
      shared[4 + threadIdx.x / 64] = l;
    }
    __syncthreads();
    top = fmaxf(fmaxf(shared[0], shared[1]), fmaxf(shared[2], shared[3]));
    least = -fmaxf(fmaxf(shared[4], shared[5]), fmaxf(shared[6], shared[7]));
  }
};

// ── even blocks ─────────────────────────────────────────────────────────────
// A number of a cut block is off by up to 2^-22 of itself or 2^-40 of the block's
// largest, whichever is more, and probabilities and gradients of scores are cut
// at 2^-37 of what they can be at most. So where rows or columns are of very
// unlike sizes, float32 would keep of the small ones what this loses, and a
// key that a query does not even see would set the scale of those it sees. The
// launches that cut operands write how even each block is, and workgroups that
// meet blocks (or scores, or sizes of blocks) beyond these bounds take float32
// matrix products of the operands as they are instead:
//   rows of all values, of all keys (dq) and of all queries (dk), to the largest:
//   2^-37 of a probability is then 2^-27 of what the least row adds;
constexpr int kSpread = 10;
//   rows of one block of g': gradients of scores are cut at 2^-24 of the least;
constexpr int kGradRowSpread = 13;
//   blocks of g': the sums of dv and dk follow each block's scale, but 60 at most;
constexpr int kGradSpread = 40;
//   columns of one block (one row alone is a column each, so no less), or more
//   than a sixteenth of its numbers 2^-kSmall of the largest;
constexpr int kColumnSpread = 20, kSmall = 16;
//   scores: 2^-40 of the largest is 2^-20, half a step of a float32 score of 16.
constexpr int kMostScore = 20;
constexpr int kNoRange = 1000;  // beyond every power of two of a float, up or down
constexpr int kUneven = 4096;   // added to an exponent: the block is uneven in itself

// How even a block is: the power of two above its largest number, and minus
// that of its smallest row that is not zero (kNoRange more where its columns
// or too many of its numbers are small). Both are least for a block of zeros,
// and both beyond every bound for one that is not finite, so that blocks taken
// together have the largest of each.
typedef short Range __attribute__((ext_vector_type(2)));
constexpr int kNotFinite = 8 * kNoRange;

__device__ inline Range no_range() { return Range{static_cast<short>(-kNoRange), static_cast<short>(-kNoRange)}; }
__device__ inline Range widest(Range a, Range b) { return __builtin_elementwise_max(a, b); }
__device__ inline int spread(Range r) { return r[0] + r[1]; }
// Whether a block of queries, or of their gradients, is uneven in itself.
__device__ inline bool uneven_in_itself(Range r, bool grads) { return spread(r) > (grads ? kGradRowSpread : kSpread); }
// A block's range without its rows': what its largest number spreads over blocks.
__device__ inline Range top_only(Range r) { return r[0] == -kNoRange ? r : Range{r[0], static_cast<short>(-r[0])}; }

// The range of one number.
__device__ inline Range top_range(float top) {
  if (top == 0.f) return no_range();
  if (!(top < INFINITY)) return Range{static_cast<short>(kNotFinite), static_cast<short>(kNotFinite)};
  int e;
  frexpf(top, &e);
  return Range{static_cast<short>(e), static_cast<short>(-e)};
}

// The widest of a wave's lanes, in scalar registers.
__device__ inline Range wave_widest(Range r) {
  const int x = join_wave(__builtin_bit_cast(int, r), [](int a, int b) {
    return __builtin_bit_cast(int, widest(__builtin_bit_cast(Range, a), __builtin_bit_cast(Range, b)));
  });
  return __builtin_bit_cast(Range, __builtin_amdgcn_readfirstlane(x));
}

// Two matrices' ranges: of keys and values, or of queries and gradients.
struct Ranges {
  Range first, second;
};

// The widest of `n` blocks, for a whole wave.
__device__ inline Ranges widest_of(const Ranges* ranges, int n) {
  Ranges r = {no_range(), no_range()};
  for (int i = threadIdx.x % 64; i < n; i += 64) {
    const Ranges b = ranges[i];
    r.first = widest(r.first, b.first);
    r.second = widest(r.second, b.second);
  }
  return {wave_widest(r.first), wave_widest(r.second)};
}

// ... of the blocks' largest numbers alone, and whether any is uneven in itself.
struct Tops {
  Range first, second;
  bool uneven;
};
__device__ inline Tops tops_of(const Ranges* ranges, int n) {
  Tops r = {no_range(), no_range(), false};
  for (int i = threadIdx.x % 64; i < n; i += 64) {
    const Ranges b = ranges[i];
    r.first = widest(r.first, top_only(b.first));
    r.second = widest(r.second, top_only(b.second));
    r.uneven |= uneven_in_itself(b.first, false) || uneven_in_itself(b.second, true);
  }
  return {wave_widest(r.first), wave_widest(r.second), __any(r.uneven) != 0};
}

// The power of two above |scale| log2 e D: what the largest numbers of a query
// and a key are multiplied by to bound their score.
__device__ inline int score_exponent(float scale, int D) {
  int e;
  frexpf(fabsf(scale) * kLog2e * D, &e);
  return e;
}

// The range of a block in LDS, in the threads of the first wave. `top` and
// `least` are its largest magnitude and its smallest that is not zero, in all
// threads; every thread takes part. Where no number is 2^-kColumnSpread of the
// largest, nor is a column (nearly all blocks of numbers drawn alike), and only
// its rows are looked at: the launches that cut operands took up to 4 us more
// with the columns of every block looked at.
struct RangeSpace {
  float lows[4], columns[256];
  int counts[4];
};
template <int NB>
__device__ inline Range block_range(const float* x, float top, float least, RangeSpace& shared, int D) {
  const int wave = threadIdx.x / 64, row = threadIdx.x / 8, part = threadIdx.x % 8 * 4;
  float of_row = 0.f;
#pragma unroll
  for (int n = 0; n < NB; n++) {
    const float4 v = *reinterpret_cast<const float4*>(x + row * kStride<NB> + 32 * n + part);
    of_row = fmaxf(of_row, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
  }
  of_row = __int_as_float(join8(__float_as_int(of_row), max_of_floats));
  int e;
  frexpf(of_row, &e);
  const float low = wave_max(of_row > 0.f ? static_cast<float>(-e) : -kNoRange);
  if (threadIdx.x % 64 == 0) shared.lows[wave] = low;
  bool uneven = false;
  if (least < ldexpf(top, -kColumnSpread)) {
    // A thread has a column's rows of its slice.
    constexpr int kColumns = NB * 32, kSlices = NB == 3 ? 2 : 256 / kColumns, kRows = 32 / kSlices;
    const int column = threadIdx.x % kColumns, slice = threadIdx.x / kColumns;
    float of_column = 0.f;
    int small = 0;
    if (slice < kSlices)
      for (int i = 0; i < kRows; i++) {
        const float a = fabsf(x[(slice * kRows + i) * kStride<NB> + column]);
        of_column = fmaxf(of_column, a);
        small += a > 0.f && a < ldexpf(top, -kSmall) ? 1 : 0;
      }
    shared.columns[threadIdx.x] = of_column;
    small = join_wave(small, [](int a, int b) { return a + b; });
    if (threadIdx.x % 64 == 0) shared.counts[wave] = small;
    __syncthreads();
    if (wave == 0) {
      for (int c = threadIdx.x; c < kColumns; c += 64) {
        float most = 0.f;
        for (int i = 0; i < kSlices; i++) most = fmaxf(most, shared.columns[i * kColumns + c]);
        uneven |= most > 0.f && most < ldexpf(top, -kColumnSpread);
      }
      uneven = __any(uneven) || shared.counts[0] + shared.counts[1] + shared.counts[2] + shared.counts[3] > 2 * D;
    }
  } else {
    __syncthreads();
  }
  if (wave > 0) return no_range();
  const float lows = fmaxf(fmaxf(shared.lows[0], shared.lows[1]), fmaxf(shared.lows[2], shared.lows[3]));
  const Range r = top_range(top);
  if (r[0] == -kNoRange || r[0] == kNotFinite) return r;
  return Range{r[0], static_cast<short>(uneven ? kNoRange : static_cast<int>(lows))};
}

// Four numbers of a row, which starts on any float: odd head sizes take the
// same 16-byte loads and stores. (As single floats a token over 8 x 8192 keys of
// 63 columns took 80 us, of 127 251; so 29 and 77, as 64 and 128 do.)
typedef float floatu4 __attribute__((ext_vector_type(4), aligned(4)));

// Columns c .. c + 3 of a row of D >= 4, or the row's last four where those would
// pass its end; `turn_to` then moves them to their places.
__device__ inline float4 load4_within(const float* row, int c, int D) {
  const floatu4 v = *reinterpret_cast<const floatu4*>(row + min(c, D - 4));
  return make_float4(v[0], v[1], v[2], v[3]);
}

// The columns past the end are then any of the row's own.
__device__ inline float4 turn_to(float4 v, int c, int D) {
  const int by = c - (D - 4);
  if (by > 0 && by & 1) v = make_float4(v.y, v.z, v.w, v.w);
  if (by > 0 && by & 2) v = make_float4(v.z, v.w, v.w, v.w);
  return v;
}

// Columns c .. c + 3 of a row of D, 0 past its end. Every lane loads from the
// row whatever it keeps: loads under conditions would wait for one another.
__device__ inline float4 load4(const float* row, int c, int D) {
  float4 v;
  if (D >= 4) v = turn_to(load4_within(row, c, D), c, D);
  else v = make_float4(row[c < D ? c : 0], row[c + 1 < D ? c + 1 : 0], row[c + 2 < D ? c + 2 : 0], 0.f);
  if (c >= D) v.x = 0.f;
  if (c + 1 >= D) v.y = 0.f;
  if (c + 2 >= D) v.z = 0.f;
  if (c + 3 >= D) v.w = 0.f;
  return v;
}

// A block of up to 32 rows of `rows` rows of D numbers into LDS, the rest 0; the
// extremes of this thread's.
template <int NB>
__device__ inline Extremes load_block(const float* src, size_t stride, int rows, int D, float* x) {
  Extremes of;
  float4 loaded[NB];
#pragma unroll
  for (int n = 0; n < NB; n++) {
    const int at = n * 256 + threadIdx.x;
    loaded[n] = load4(src + min(at / (NB * 8), rows - 1) * stride, at % (NB * 8) * 4, D);
  }
#pragma unroll
  for (int n = 0; n < NB; n++) {
    const int at = n * 256 + threadIdx.x, row = at / (NB * 8), c = at % (NB * 8) * 4;
    const float4 v = row < rows ? loaded[n] : make_float4(0.f, 0.f, 0.f, 0.f);
    of.take(v);
    *reinterpret_cast<float4*>(x + row * kStride<NB> + c) = v;
  }
  return of;
}

// The forward pass's workspace: per batch and key head and block of 32 keys the
// tile [K rows | V columns | exponents of K, V]; then the blocks' ranges; then
// the parts, where there is more than one.
template <int NB>
constexpr int kForwardTile = kRowBytes<NB> + kColBytes<NB> + kTail;

template <int NB>
__device__ inline Ranges* forward_ranges(char* ws, size_t key_blocks) {
  return reinterpret_cast<Ranges*>(ws + key_blocks * kForwardTile<NB>);
}

// Keys and values cut once per call: one workgroup per block and matrix.
// Every query tile of a head reads them, so the main loop only copies.
template <int NB>
__device__ inline void pack_keys(const float* k, const float* v, const int* lengths, char* ws, int B, int Sk, int Hk,
                                 int D) {
  __shared__ __attribute__((aligned(16))) float x[kBlock * kStride<NB>];
  __shared__ float tops[8];
  __shared__ RangeSpace ranges;
  const int blocks = (Sk + kBlock - 1) / kBlock;
  const bool values = blockIdx.x % 2;
  const size_t block = blockIdx.x / 2;  // (b, hk, kb)
  const int kb = block % blocks, hk = block / blocks % Hk, b = block / blocks / Hk;
  const int keys = lengths ? min(max(lengths[b], 0), Sk) : Sk;
  if (kb * kBlock >= keys) return;
  const size_t at = (static_cast<size_t>(b) * Sk + kb * kBlock) * Hk * D + static_cast<size_t>(hk) * D;
  Extremes of = load_block<NB>((values ? v : k) + at, static_cast<size_t>(Hk) * D, min(kBlock, keys - kb * kBlock), D, x);
  of.join(tops);
  const int e = block_exponent(of.top);
  const float scale = block_scale(e);
  char* tile = ws + block * kForwardTile<NB>;
  // Keys are multiplied into scores, which only their largest number bounds.
  const Range range = values ? block_range<NB>(x, of.top, of.least, ranges, D) : top_range(of.top);
  if (values) write_cols<NB>(x, scale, tile + kRowBytes<NB>);
  else write_rows<NB>(x, scale, tile);
  if (threadIdx.x == 0) {
    reinterpret_cast<int*>(tile + kRowBytes<NB> + kColBytes<NB>)[values] = e;
    Range* of_block = &forward_ranges<NB>(ws, static_cast<size_t>(B) * Hk * blocks)[block].first;
    of_block[values] = range;
  }
}

// Copies `Bytes` (a multiple of 1 KiB), contiguous, into LDS without passing
// registers: each wave 1 KiB at a time.
template <int Bytes, int Waves>
__device__ inline void copy_tile(const char* from, char* to) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
#pragma unroll
  for (int at = wave * kPart; at < Bytes; at += Waves * kPart)
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void*)(from + at + lane * 16),
        (__attribute__((address_space(3))) void*)(to + at), 16, 0, 0);
}

__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The copies are in LDS, and every wave is done with what it read.
__device__ inline void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// Scales of accumulators. Sums over rows meet blocks of one exponent after
// another, and accumulators hold their sums times 2^(ref): ref follows the
// blocks where they differ by more than kSlack, and results are multiplied
// up or down, exactly. It stays within 60 of the least exponent met (of the
// largest values), which keeps the sums finite.
constexpr int kSlack = 4;
struct RunningScale {
  int ref = 0, least = 0;
  bool any = false;
  // Takes block exponent e; returns the power of two that accumulators have
  // to be multiplied by (0: none), and leaves in *behind how far the block's
  // operand is above ref (what the other operand makes up for). A block of zeros
  // changes nothing: were its exponent a scale like any other, probabilities
  // would be cut to meet it, and their row's sum with them.
  __device__ int take(int e, int* behind) {
    int change = 0;
    *behind = 0;
    if (e >= kNoExponent) return 0;
    if (!any) {
      any = true;
      ref = least = e;
    } else if (e < ref || e > ref + kSlack) {
      least = min(least, e);
      const int to = min(e, least + 60);
      change = to - ref;
      ref = to;
    }
    *behind = e - ref;
    return change;
  }
};

// Probabilities are kept below 2^kLazy of 1 (the row's maximum follows only
// where it grew by more), and times 2^kProbShift, less than 2^15, when cut.
constexpr float kLazy = 2.f;
constexpr int kProbShift = 13;

// p[0..7] as two parts, cut off (not rounded: one instruction for two
// numbers), the second from what the first leaves: low by up to 2^-21 of each, or
// by 2^-37 of the largest a row can have. So what a key takes that every query
// weighs less than 2^-27 keeps fewer bits than float32's, by up to that.
__device__ inline void cut_probs(const float* p, half8* hi, half8* lo) {
  typedef __fp16 fp16x2 __attribute__((ext_vector_type(2)));
  union {
    fp16x2 two[4];
    half8 all;
  } h, l;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    h.two[i] = __builtin_amdgcn_cvt_pkrtz(p[2 * i], p[2 * i + 1]);
    l.two[i] = __builtin_amdgcn_cvt_pkrtz(p[2 * i] - static_cast<float>(h.two[i][0]),
                                          p[2 * i + 1] - static_cast<float>(h.two[i][1]));
  }
  *hi = h.all;
  *lo = l.all;
}

// Row l % 32 of this wave's 32 rows (a row to load from, also where it is not
// live and counts as 0) as the fragments of a product over its
// columns, times `times` and sign 2^e with an exponent of the row's own.
template <int NB>
__device__ inline int row_fragments(const float* row, bool live, int D, float sign, float times, half8 (&hi)[NB * 2],
                                    half8 (&lo)[NB * 2]) {
  const int half = threadIdx.x % 64 / 32;
  float v[NB * 2][8];
  float top = 0.f;
#pragma unroll
  for (int t = 0; t < NB * 2; t++)
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float4 x = load4(row, 16 * t + 8 * half + i, D);
      v[t][i] = x.x;
      v[t][i + 1] = x.y;
      v[t][i + 2] = x.z;
      v[t][i + 3] = x.w;
    }
#pragma unroll
  for (int t = 0; t < NB * 2; t++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      v[t][i] = live ? v[t][i] * times : 0.f;
      top = v[t][i] == v[t][i] ? fmaxf(top, fabsf(v[t][i])) : INFINITY;
    }
  const int e = block_exponent(halves_max(top));
  const float scale = sign * block_scale(e);
#pragma unroll
  for (int t = 0; t < NB * 2; t++) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[t][i] *= scale;
    cut(v[t], &hi[t], &lo[t]);
  }
  return e;
}

// 16 result registers of a 32-column group of row `row`: columns 32 n +
// result_row(r, half), times scale 2^e (the power last: alone it may be out of
// range).
__device__ inline void store_columns(float* row, int n, int half, int D, const floatx16& o, float scale, int e) {
#pragma unroll
  for (int g = 0; g < 4; g++) {
    const int c = 32 * n + 8 * g + 4 * half;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = ldexpf(o[4 * g + i] * scale, e);
    if (c + 3 < D) {
      *reinterpret_cast<floatu4*>(row + c) = floatu4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (c + i < D) row[c + i] = v[i];
    }
  }
}

// ── products in float32 ─────────────────────────────────────────────────────
// What uneven operands take: float32 matrix products of 32 x 32 x 2, with
// operands loaded as they are, by waves that share nothing. Lane l has row (or
// column) l % 32 of an operand and terms 4 (l / 32) .. + 3 of every eight; results
// lie as those of cut operands do. Right, not fast, in as few registers as the
// loops over even blocks leave: with one value 10^8 times the others 4096 causal
// tokens, 32 heads of 128 over 8, take 2.4 ms instead of 0.4, and 8192 with
// gradients, 16 heads over 4, 34 ms instead of 3.4; with such a gradient in every
// 20th block of queries 11 ms. Looking for it costs even operands 0 to 5 in 100.

// The kernel's arguments, read again: held in registers through the loops over
// even blocks they would be spilled there.
struct ForwardArgs {
  float* y;
  const float *q, *k, *v;
};
struct GradArgs {
  float* dq;
  const float *q, *k, *v, *y, *g, *stats;
};
template <class Args>
__device__ inline const Args* args_again() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return (const Args*)p;  // of the constant address space
}

// Products of two rows of D numbers.
template <int NB>
__device__ inline floatx16 exact_dots(const float* a, const float* b, int D) {
  const int half = threadIdx.x % 64 / 32;
  floatx16 x = {};
#pragma unroll 1
  for (int c = 4 * half; c < NB * 32; c += 8) {
    const float4 av = load4(a, c, D), bv = load4(b, c, D);
    x = __builtin_amdgcn_mfma_f32_32x32x2f32(av.x, bv.x, x, 0, 0, 0);
    x = __builtin_amdgcn_mfma_f32_32x32x2f32(av.y, bv.y, x, 0, 0, 0);
    x = __builtin_amdgcn_mfma_f32_32x32x2f32(av.z, bv.z, x, 0, 0, 0);
    x = __builtin_amdgcn_mfma_f32_32x32x2f32(av.w, bv.w, x, 0, 0, 0);
  }
  return x;
}

// o += X^T p with the first `rows` of 32 rows of X, multiplied by `times(row)`
// 2^e, and p as a product leaves it: 0 for the rows past them, for which the
// last is read again. Columns past D are any.
template <int NB, class Times>
__device__ inline void exact_outer(floatx16 (&o)[NB], const float* x, size_t stride, int rows, int D, const floatx16& p,
                                   int e, Times times) {
  const int column = threadIdx.x % 32, half = threadIdx.x % 64 / 32;
  asm volatile("" : "+s"(rows));  // or the caller's sixteen numbers of rows stay in registers
#pragma unroll
  for (int r = 0; r < 16; r++) {
    const int row = result_row(r, half);
    const float* at = x + min(row, rows - 1) * stride;
    const float by = times(min(row, rows - 1));
#pragma unroll
    for (int n = 0; n < NB; n++)
      o[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(ldexpf(at[min(32 * n + column, D - 1)] * by, e), p[r], o[n], 0, 0, 0);
    // Few loads in flight, so that even blocks have no fewer registers for these.
    if (r % 2) __builtin_amdgcn_sched_barrier(0);
  }
}

// ── keys in parts ───────────────────────────────────────────────────────────
// Where the query rows alone are too few workgroups, each takes a part of the
// keys and leaves, per row (b, h, i), the sum of exp2(S_ij log2 e - m) v_j, m,
// and the sum of the exponentials (0: it saw no key, and the rest is nothing).
struct RowParts {
  float* ml;  // [split][row][2]: first, so that pairs are on the alignment of pairs whatever D
  float* o;   // [split][row][D]
  size_t rows;
};

__device__ inline RowParts row_parts(char* at, const Shape& s, int splits) {
  RowParts p;
  p.rows = static_cast<size_t>(s.b) * s.hq * s.sq;
  p.ml = reinterpret_cast<float*>(at);
  p.o = p.ml + 2 * splits * p.rows;
  return p;
}

// Keys a part where all sequences' keys go into about `units` parts of the same
// length, no more than `splits` of a sequence: where lengths differ a short
// sequence takes few workgroups, and all of them end together. For up to 64
// sequences; lane l has sequence l's keys.
__device__ inline unsigned keys_a_part(const Shape& s, int keys, int splits, int units) {
  unsigned all = (keys + 63u) / 64;  // in 64 keys, of which a wave takes 16
  for (int d = 32; d > 0; d /= 2) all += __shfl_xor(all, d);
  const unsigned longest = (s.sk + 63u) / 64;
  return __builtin_amdgcn_readfirstlane(64 * max(max((all + units - 1) / units, (longest + splits - 1) / splits), 2u));
}

// The parts joined: a thread per row and W columns, N parts at a time in flight.
// Where a row is no whole number of W its last thread takes its last W columns,
// some of them a second time. The stats are written by the row's first column.
template <int N, int W, bool OneLength>
__device__ inline void join_columns(float* __restrict__ y, float* __restrict__ stats, const int* __restrict__ lengths,
                                    const RowParts& parts, const Shape& s, int splits, int units) {
  int each = 0;
  if (OneLength) {
    const int lane = threadIdx.x % 64;
    each = keys_a_part(s, lane < s.b ? key_count(s, lengths, lane) : 0, splits, units);
  }
  const size_t e = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  const int columns = (s.d + W - 1) / W;
  if (e >= parts.rows * columns) return;
  const size_t row = e / columns;
  const int d = min(static_cast<int>(e % columns) * W, s.d - W);
  const int i = row % s.sq, h = row / s.sq % s.hq;
  const size_t b = row / s.sq / s.hq;
  if (OneLength) splits = (static_cast<unsigned>(key_count(s, lengths, b)) + each - 1) / each;
  float top = -INFINITY, sum = 0.f, all[W] = {};
  for (int p0 = 0; p0 < splits; p0 += N) {
    float2 ml[N];
    float o[N][W];
#pragma unroll
    for (int n = 0; n < N; n++) {
      const size_t part = min(p0 + n, splits - 1) * parts.rows + row;
      ml[n] = *reinterpret_cast<const float2*>(parts.ml + 2 * part);
      if constexpr (W == 4) {
        const floatu4 v = *reinterpret_cast<const floatu4*>(parts.o + part * s.d + d);
#pragma unroll
        for (int w = 0; w < 4; w++) o[n][w] = v[w];
      } else {
        o[n][0] = parts.o[part * s.d + d];
      }
    }
    float most = top;
#pragma unroll
    for (int n = 0; n < N; n++) {
      if (p0 + n >= splits) ml[n].y = 0.f;
      if (ml[n].y != 0.f) most = fmaxf(most, ml[n].x);
    }
    // A part whose sum is NaN counts: only 0 says that it saw no key.
    const float base = most == -INFINITY ? 0.f : most, old = exp2f(top - base);
    sum *= old;
#pragma unroll
    for (int w = 0; w < W; w++) all[w] *= old;
    top = most;
#pragma unroll
    for (int n = 0; n < N; n++)
      if (ml[n].y != 0.f) {
        const float of = exp2f(ml[n].x - base);
        sum += of * ml[n].y;
#pragma unroll
        for (int w = 0; w < W; w++) all[w] += of * o[n][w];
      }
  }
  const float inv = inverse_sum(sum);
  float* out = y + (b * s.sq + i) * s.hq * s.d + static_cast<size_t>(h) * s.d + d;
#pragma unroll
  for (int w = 0; w < W; w++) all[w] *= inv;
  if constexpr (W == 4) *reinterpret_cast<floatu4*>(out) = floatu4{all[0], all[1], all[2], all[3]};
  else *out = all[0];
  if (d == 0) {
    stats[row] = top == -INFINITY ? 0.f : top;
    stats[parts.rows + row] = inv;
  }
}

template <int W, bool OneLength>
__device__ inline void join_parts(float* __restrict__ y, float* __restrict__ stats, const int* __restrict__ lengths,
                                  char* __restrict__ at, const Shape& s, int splits, int units) {
  const RowParts parts = row_parts(at, s, splits);
  if constexpr (OneLength) join_columns<16, W, true>(y, stats, lengths, parts, s, splits, units);
  else if (splits <= 4) join_columns<4, W, false>(y, stats, lengths, parts, s, splits, units);
  else join_columns<16, W, false>(y, stats, lengths, parts, s, splits, units);
}

// Which `rows` queries, head, batch and part of the keys a workgroup takes. The
// last queries of every head come first: with `causal` they see the most keys,
// and what is left for the end is small. Workgroups go to the 8 chiplets in turn, so
// where the heads allow it each chiplet gets heads next to each other, which
// share keys in its cache.
__device__ inline void query_tile(const Shape& s, int rows, int splits, unsigned block, int* qt, int* h, int* b, int* split) {
  const unsigned heads = static_cast<unsigned>(s.b) * s.hq, tiles = (s.sq + rows - 1) / rows;
  unsigned head = block % heads;
  if (heads % 8 == 0) head = head % 8 * (heads / 8) + head / 8;
  *split = block / heads % splits;
  *qt = tiles - 1 - block / heads / splits;
  *h = head % s.hq;
  *b = head / s.hq;
}

// A workgroup: 128 queries of one head, 32 a wave; all keys, 32 at a time.
// S^T = K Q^T, so that a lane holds 16 scores of one query: the row's maximum
// and sum cost one exchange between the wave's halves, and the probabilities
// are in registers what O^T += V^T P^T takes as its second operand.
//
// 4096 causal tokens, 32 heads of 128 over 8: 407 us, 1013 TFLOP/s of float16
// products (338 of the float32 ones they stand for; float32's own matrix rate is
// 152 and a library's large float16 product reaches 1084). Nothing is at its
// limit: the matrix cores are busy 58% of the cycles in which a compute unit has
// waves, and waves wait 43% of theirs, for tiles and for results, at 1.9 GHz of
// 2.4, which the power leaves. Four waves a workgroup and two workgroups a compute
// unit, so that one has the cores while the other makes its probabilities; keys
// are cut by a launch of their own (15 us), once for all the query tiles that read
// them.
template <int NB>
__device__ inline void forward_tiles(float* __restrict__ y, const float* __restrict__ q, float* __restrict__ stats,
                                     const int* __restrict__ lengths, char* __restrict__ ws, const Shape& s, float scale,
                                     int splits) {
  constexpr int kTile = kForwardTile<NB>;
  // Two buffers of their own, and a loop written out twice: the compiler then
  // knows that what a step reads is not what its copies write, and does not
  // wait for them first.
  __shared__ __attribute__((aligned(1024))) char even[kTile], odd[kTile];
  __shared__ int uneven[4];
  int qt, h, b, split;
  query_tile(s, 128, splits, blockIdx.x, &qt, &h, &b, &split);
  const int hk = h / (s.hq / s.hk);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, half = lane / 32;
  const int i = qt * 128 + wave * 32 + lane % 32;  // this lane's query
  const bool live = i < s.sq;
  const int keys = key_count(s, lengths, b), first = qt * 128 + wave * 32;
  // Blocks of keys that the last query of the workgroup sees, of which this
  // part takes those from `begin` to `end`; those that the last of the wave
  // sees; those that every query of the wave sees whole.
  const int blocks = (visible(s, keys, min(s.sq, qt * 128 + 128) - 1) + kBlock - 1) / kBlock;
  const int begin = static_cast<int>(static_cast<long long>(blocks) * split / splits);
  const int end = static_cast<int>(static_cast<long long>(blocks) * (split + 1) / splits);
  const int wave_end = first < s.sq ? (visible(s, keys, min(s.sq, first + 32) - 1) + kBlock - 1) / kBlock : 0;
  const int wave_full = visible(s, keys, first) / kBlock;
  const int seen = live ? visible(s, keys, i) : 0;

  const size_t head = static_cast<size_t>(b) * s.hk + hk, head_blocks = (s.sk + kBlock - 1) / kBlock;
  const char* tile = ws + head * head_blocks * kTile;
  if (begin < end) copy_tile<kTile, 4>(tile + static_cast<size_t>(begin) * kTile, even);

  const size_t tiles = static_cast<size_t>(s.b) * s.hk * head_blocks;
  const float* q_row = q + (static_cast<size_t>(b) * s.sq + min(i, s.sq - 1)) * s.hq * s.d + static_cast<size_t>(h) * s.d;
  half8 qh[NB * 2], ql[NB * 2];
  const int eq = row_fragments<NB>(q_row, live, s.d, scale < 0.f ? -1.f : 1.f, 1.f, qh, ql);
  const Ranges seen_keys = widest_of(forward_ranges<NB>(ws, tiles) + head * head_blocks, blocks);
  if (lane == 0) uneven[wave] = 0;
  // The query's largest number is below 2^(15 - eq).
  if (__any(eq < kNoExponent && 15 - eq + seen_keys.first[0] + score_exponent(scale, s.d) > kMostScore) ||
      spread(seen_keys.second) > kSpread)
    uneven[wave] = 1;
  const float factor = fabsf(scale) * kLog2e;
  float m = -INFINITY, l = 0.f;
  floatx16 o[NB] = {};
  RunningScale vs;
  tile_barrier();
  const bool exact = uniform(uneven[0] | uneven[1] | uneven[2] | uneven[3]) != 0;
  auto finish = [&](int exponent) {
    l = halves_sum(l);
    if (!live) return;
    const size_t stat = (static_cast<size_t>(b) * s.hq + h) * s.sq + i, rows = static_cast<size_t>(s.b) * s.hq * s.sq;
    if (splits > 1) {
      const RowParts parts = row_parts(reinterpret_cast<char*>(forward_ranges<NB>(ws, tiles) + tiles), s, splits);
      const size_t out = split * rows + stat;
#pragma unroll
      for (int n = 0; n < NB; n++) store_columns(parts.o + out * s.d, n, half, s.d, o[n], 1.f, exponent);
      if (half == 0) {
        parts.ml[2 * out] = m;
        parts.ml[2 * out + 1] = l;
      }
      return;
    }
    const float inv = inverse_sum(l);
    float* row = y + (static_cast<size_t>(b) * s.sq + i) * s.hq * s.d + static_cast<size_t>(h) * s.d;
#pragma unroll
    for (int n = 0; n < NB; n++) store_columns(row, n, half, s.d, o[n], inv, exponent);
    if (half == 0) {
      stats[stat] = m == -INFINITY ? 0.f : m;
      stats[rows + stat] = inv;
    }
  };
  if (__builtin_expect(exact, 0)) {
    const size_t stride = static_cast<size_t>(s.hk) * s.d, of_head = static_cast<size_t>(b) * s.sk * stride + static_cast<size_t>(hk) * s.d;
    const auto* again = args_again<ForwardArgs>();
    const float *k = again->k, *v = again->v;
    for (int kb = begin; kb < min(end, wave_end); kb++) {
      const size_t at = of_head + static_cast<size_t>(kb) * kBlock * stride;
      const int rows = min(kBlock, keys - kb * kBlock);
      floatx16 x = exact_dots<NB>(k + at + min(lane % 32, rows - 1) * stride, q_row, s.d);
      float top = m;
#pragma unroll
      for (int r = 0; r < 16; r++) {
        x[r] = kb * kBlock + result_row(r, half) < seen ? x[r] * (scale * kLog2e) : -INFINITY;
        top = fmaxf(top, x[r]);
      }
      top = halves_max(top);
      const float base = top == -INFINITY ? 0.f : top, old = exp2f(m - base);
      m = top;
      l *= old;
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[n][r] *= old;
#pragma unroll
      for (int r = 0; r < 16; r++) {
        x[r] = exp2f(x[r] - base);
        l += x[r];
      }
      exact_outer<NB>(o, v + at, stride, rows, s.d, x, 0, [](int) { return 1.f; });
    }
    finish(0);
    return;
  }
  auto step = [&](const char* now, char* next, int kb) {
    if (kb + 1 < end) copy_tile<kTile, 4>(tile + static_cast<size_t>(kb + 1) * kTile, next);
    if (kb < wave_end) {
      const char* t = now + lane * 16;
      const int* tail = reinterpret_cast<const int*>(now + kTile - kTail);
      const int ek = uniform(tail[0]), ev = uniform(tail[1]);
      floatx16 x = {};
#pragma unroll
      for (int n = 0; n < NB * 2; n++)
        x = mfma3(*reinterpret_cast<const half8*>(t + n * 2 * kPart), *reinterpret_cast<const half8*>(t + n * 2 * kPart + kPart),
                  qh[n], ql[n], x);
      float fac = ldexpf(factor, -(eq + ek));
      if (kb >= wave_full) {
#pragma unroll
        for (int r = 0; r < 16; r++) x[r] = kb * kBlock + result_row(r, half) < seen ? x[r] * fac : -INFINITY;
        fac = 1.f;
      }
      float top = x[0];
#pragma unroll
      for (int r = 1; r < 16; r++) top = fmaxf(top, x[r]);
      top = halves_max(top) * fac;
      int behind;
      const int change = vs.take(ev, &behind);
      if (change != 0) {
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
          for (int r = 0; r < 16; r++) o[n][r] = ldexpf(o[n][r], change);
      }
      if (__any(top > m + kLazy)) {
        const float to = top > m + kLazy ? top : m;
        const float old = to == -INFINITY ? 1.f : exp2f(m - to);
        m = to;
        l *= old;
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
          for (int r = 0; r < 16; r++) o[n][r] *= old;
      }
      // p 2^(13 - behind): what the block's values are above ref goes off here.
      const float base = static_cast<float>(kProbShift - behind) - (m == -INFINITY ? 0.f : m);
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; r++) {
        x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], fac, base));
        sum += x[r];
      }
      l += ldexpf(sum, behind - kProbShift);
#pragma unroll
      for (int u = 0; u < 2; u++) {
        float p[8];
#pragma unroll
        for (int r = 0; r < 8; r++) p[r] = x[8 * u + r];
        half8 ph, pl;
        cut_probs(p, &ph, &pl);
        const char* vt = t + kRowBytes<NB> + u * 2 * kPart;
#pragma unroll
        for (int n = 0; n < NB; n++)
          o[n] = mfma3(*reinterpret_cast<const half8*>(vt + n * 4 * kPart),
                       *reinterpret_cast<const half8*>(vt + n * 4 * kPart + kPart), ph, pl, o[n]);
      }
    }
    tile_barrier();
  };
  for (int kb = begin; kb < end; kb += 2) {
    step(even, odd, kb);
    if (kb + 1 < end) step(odd, even, kb + 1);
  }
  finish(-kProbShift - vs.ref);
}

// ── gradients ───────────────────────────────────────────────────────────────
// With r_i = 1 / (row i's sum), p_ij = exp2(S_ij log2 e - m_i) (r_i p_ij is the
// probability), g'_i = r_i g_i and delta_i = g'_i . y_i:
//   dv_j = sum_i p_ij g'_i
//   ds_ij = p_ij (g'_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
// so that both p and ds are cut where their largest is, whatever the row's sum.
// |g'_i . v_j - delta_i| is at most twice |g'_i| times the largest |v_j| that i
// sees, and p less than 2^kLazy: ds times 2^(kScoreShift - the norms' exponents)
// is less than 2^15, with the largest |g'_i| of the block and the largest |v_j|
// that the workgroup's queries see (dq) or of the head (dk).
constexpr int kScoreShift = 12;  // 15, less kLazy and one for the twice

// The gradients' workspace. Per batch and key head and block of 32 keys: the
// tile [K rows | V rows | K columns | exponents of K, V]; per batch and query
// head and block of 32 queries: the tile [Q rows | G rows | Q columns | G
// columns | m, delta of each row, exponents of Q, G (kUneven more where the block
// is uneven in itself) and of G's largest row norm] (G = g'); then the ranges of
// the key blocks and of the query blocks; then the exponents of the key blocks'
// largest row norms of V; then dk and dv of each part of the queries, and dq of each part of the keys,
// where there is more than one.
template <int NB>
constexpr int kKeyTile = 2 * kRowBytes<NB> + kColBytes<NB> + kTail;
template <int NB>
constexpr int kQueryTile = 2 * kRowBytes<NB> + 2 * kColBytes<NB> + kTail;

struct GradSpace {
  int k_blocks, q_blocks;
  char *k_tiles, *q_tiles;
  Ranges *k_ranges, *q_ranges;
  int* norms;
  float* parts;
};

template <int NB>
__device__ inline GradSpace grad_space(char* ws, const Shape& s) {
  GradSpace g;
  g.k_blocks = (s.sk + kBlock - 1) / kBlock;
  g.q_blocks = (s.sq + kBlock - 1) / kBlock;
  const size_t nk = static_cast<size_t>(s.b) * s.hk * g.k_blocks, nq = static_cast<size_t>(s.b) * s.hq * g.q_blocks;
  g.k_tiles = ws;
  g.q_tiles = ws + nk * kKeyTile<NB>;
  g.k_ranges = reinterpret_cast<Ranges*>(g.q_tiles + nq * kQueryTile<NB>);
  g.q_ranges = g.k_ranges + nk;
  g.norms = reinterpret_cast<int*>(g.q_ranges + nq);
  g.parts = reinterpret_cast<float*>(g.norms + (nk + 3) / 4 * 4);
  return g;
}

// Floats of the parts of dk and dv.
__device__ inline size_t key_parts(const Shape& s, int parts) {
  return parts > 1 ? 2 * static_cast<size_t>(parts) * s.b * s.sk * s.hk * s.d : 0;
}

// The power of two above a norm, from the largest sum of squares of a block's
// numbers times 2^e.
__device__ inline int norm_exponent(float squares, int e) {
  if (squares == 0.f) return -120;
  if (!(squares < INFINITY)) return 0;
  int k;
  frexpf(squares, &k);
  return max((k + 1) / 2 - e, -120);
}

// 2^a for any a, saturating.
__device__ inline float power(int a) { return ldexpf(1.f, a); }

// Keys, values, queries and gradients cut once per call, one workgroup per
// block and matrix, with how even each block is. Bound by memory: 16 heads of 128 over 8192 tokens 102 us for
// 236 MB read and 320 written, 5.4 TB/s (queries and gradients by rows for the
// scores, and by columns for dk and dv). With the outputs read after the gradients
// were in LDS it took 138.
template <int NB>
__device__ inline void pack_grad(const float* __restrict__ q, const float* __restrict__ k, const float* __restrict__ v,
                                 const float* __restrict__ y, const float* __restrict__ g,
                                 const float* __restrict__ stats, const int* __restrict__ lengths,
                                 char* __restrict__ ws, const Shape& s) {
  __shared__ __attribute__((aligned(16))) float x[kBlock * kStride<NB>];
  __shared__ float tops[8];
  __shared__ RangeSpace ranges;
  const GradSpace f = grad_space<NB>(ws, s);
  const size_t nk = static_cast<size_t>(s.b) * s.hk * f.k_blocks;
  const bool second = blockIdx.x % 2;  // V, or G
  size_t block = blockIdx.x / 2;
  const bool of_keys = block < nk;
  if (!of_keys) block -= nk;
  const int blocks = of_keys ? f.k_blocks : f.q_blocks, heads = of_keys ? s.hk : s.hq, n = of_keys ? s.sk : s.sq;
  const int at = block % blocks * kBlock, h = block / blocks % heads, b = block / blocks / heads;
  const int rows = of_keys ? key_count(s, lengths, b) : n;
  if (at >= rows) return;
  const size_t stride = static_cast<size_t>(heads) * s.d;
  const size_t first = (static_cast<size_t>(b) * n + at) * stride + static_cast<size_t>(h) * s.d;
  const float* src = (of_keys ? (second ? v : k) : (second ? g : q)) + first;
  const int row = threadIdx.x / 8, part = threadIdx.x % 8 * 4;  // eight threads a row, for its sums: columns part .. part + 3 of every 32
  const bool of_grads = !of_keys && second, live = at + row < s.sq;
  float4 yv[NB];
  float m = 0.f, inv = 0.f;
  if (of_grads) {
    const int to_load = min(row, rows - at - 1);
#pragma unroll
    for (int n = 0; n < NB; n++) yv[n] = load4(y + first + to_load * stride, 32 * n + part, s.d);
    const size_t stat = (static_cast<size_t>(b) * s.hq + h) * s.sq + at + to_load;
    m = stats[stat];
    inv = stats[static_cast<size_t>(s.b) * s.hq * s.sq + stat];
  }
  Extremes of = load_block<NB>(src, stride, min(kBlock, rows - at), s.d, x);
  char* tile = of_keys ? f.k_tiles + block * kKeyTile<NB> : f.q_tiles + block * kQueryTile<NB>;
  char* tail = tile + (of_keys ? kKeyTile<NB> : kQueryTile<NB>) - kTail;
  int* exponents = reinterpret_cast<int*>(tail) + (of_keys ? 0 : 64);
  float4* mine = reinterpret_cast<float4*>(x + row * kStride<NB> + part);  // every eighth
  if (of_grads) {
    // g' and delta; rows past the last query stay 0.
    __syncthreads();
    float delta = 0.f;
    of = Extremes();
#pragma unroll
    for (int n = 0; n < NB; n++) {
      float4 gx = mine[8 * n];
      gx = live ? make_float4(gx.x * inv, gx.y * inv, gx.z * inv, gx.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
      mine[8 * n] = gx;
      of.take(gx);
      if (live) delta += gx.x * yv[n].x + gx.y * yv[n].y + gx.z * yv[n].z + gx.w * yv[n].w;
    }
    delta = sum8(delta);
    if (part == 0) {
      reinterpret_cast<float*>(tail)[row] = live ? m : 0.f;
      reinterpret_cast<float*>(tail)[32 + row] = delta;
    }
  }
  of.join(tops);
  const int e = block_exponent(of.top);
  const float scale = block_scale(e);
  const Range range = block_range<NB>(x, of.top, of.least, ranges, s.d);
  if (second) {
    float squares = 0.f;
#pragma unroll
    for (int n = 0; n < NB; n++) {
      const float4 v = mine[8 * n];
      const float a[4] = {v.x * scale, v.y * scale, v.z * scale, v.w * scale};
#pragma unroll
      for (int i = 0; i < 4; i++) squares += a[i] * a[i];
    }
    squares = sum8(squares);
    __syncthreads();  // tops is read
    squares = block_max(squares, tops);
    if (threadIdx.x == 0) *(of_keys ? f.norms + block : exponents + 2) = norm_exponent(squares, e);
  }
  if (threadIdx.x == 0) {
    exponents[second] = e + (!of_keys && uneven_in_itself(range, second) ? kUneven : 0);
    (&(of_keys ? f.k_ranges : f.q_ranges)[block].first)[second] = range;
  }
  write_rows<NB>(x, scale, tile + (second ? kRowBytes<NB> : 0));
  if (of_keys && !second) write_cols<NB>(x, scale, tile + 2 * kRowBytes<NB>);
  if (!of_keys) write_cols<NB>(x, scale, tile + 2 * kRowBytes<NB> + (second ? kColBytes<NB> : 0));
}

// The exponent above the norms of the value rows of a head's first blocks.
__device__ inline int values_norm(const int* norms, int blocks) {
  int top = -120;
  for (int n = threadIdx.x % 64; n < blocks; n += 64) top = max(top, norms[n]);
  return __builtin_amdgcn_readfirstlane(join_wave(top, [](int a, int b) { return max(a, b); }));
}

__device__ inline int clamp_power(int a) { return min(max(a, -120), 120); }

// dq. A workgroup: 32 queries of one head a wave, over all keys; scores and
// their gradients transposed as in the forward pass. Tiles of four column
// groups leave room for one workgroup a compute unit: eight waves share them,
// so that each matrix core has two waves in turn. 16 heads of 128 over 8192 causal
// tokens: 1021-1042 us, up to 1210 TFLOP/s of float16 products, the cores busy 66%
// and waves waiting 46% of their cycles, at 1.9 GHz.
template <int NB>
constexpr int kQueryGradWaves = NB < 4 ? 4 : 8;

template <int NB, int Waves>
__device__ inline void query_grads(float* __restrict__ dq, const float* __restrict__ q, const float* __restrict__ g,
                                   const float* __restrict__ stats, const int* __restrict__ lengths,
                                   char* __restrict__ ws, const Shape& s, float scale, int parts, int q_parts,
                                   unsigned block, char* even, char* odd) {
  constexpr int kTile = kKeyTile<NB>;
  const GradSpace f = grad_space<NB>(ws, s);
  int qt, h, b, part;
  constexpr int kRows = 32 * Waves;
  query_tile(s, kRows, q_parts, block, &qt, &h, &b, &part);
  const int hk = h / (s.hq / s.hk);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, half = lane / 32;
  const int first = qt * kRows + wave * 32, i = first + lane % 32;
  const bool live = i < s.sq, wave_live = first < s.sq;
  const int keys = key_count(s, lengths, b);
  const int blocks = (visible(s, keys, min(s.sq, qt * kRows + kRows) - 1) + kBlock - 1) / kBlock;
  const int begin = static_cast<int>(static_cast<long long>(blocks) * part / q_parts);
  const int end = static_cast<int>(static_cast<long long>(blocks) * (part + 1) / q_parts);
  const int wave_end = wave_live ? (visible(s, keys, min(s.sq, first + 32) - 1) + kBlock - 1) / kBlock : 0;
  const int wave_full = visible(s, keys, first) / kBlock;
  const int seen = live ? visible(s, keys, i) : 0;

  const size_t head = static_cast<size_t>(b) * s.hk + hk;
  const char* tile = f.k_tiles + head * f.k_blocks * kTile;
  if (begin < end) copy_tile<kTile, Waves>(tile + static_cast<size_t>(begin) * kTile, even);

  const size_t at = (static_cast<size_t>(b) * s.sq + min(i, s.sq - 1)) * s.hq * s.d + static_cast<size_t>(h) * s.d;
  const size_t stat = (static_cast<size_t>(b) * s.hq + h) * s.sq + min(i, s.sq - 1);
  const size_t q_block = (static_cast<size_t>(b) * s.hq + h) * f.q_blocks + min(first / kBlock, f.q_blocks - 1);
  const float inv = live ? stats[static_cast<size_t>(s.b) * s.hq * s.sq + stat] : 0.f;
  const float m = live ? stats[stat] : 0.f;
  const char* q_tail = f.q_tiles + (q_block + 1) * kQueryTile<NB> - kTail;
  const float delta = reinterpret_cast<const float*>(q_tail)[32 + lane % 32];
  const int shift = uniform(clamp_power(kScoreShift - reinterpret_cast<const int*>(q_tail)[66] -
                                        values_norm(f.norms + head * f.k_blocks, blocks)));
  // Whether the keys and values that the workgroup's queries see and each block of
  // its own are even, and their scores small enough.
  const Ranges seen_keys = widest_of(f.k_ranges + head * f.k_blocks, blocks);
  const int own = (static_cast<size_t>(qt) * kRows) / kBlock;
  const Tops of_rows = tops_of(f.q_ranges + (static_cast<size_t>(b) * s.hq + h) * f.q_blocks + own, min(Waves, f.q_blocks - own));
  const bool exact = max(spread(seen_keys.first), spread(seen_keys.second)) > kSpread || of_rows.uneven ||
                     of_rows.first[0] + seen_keys.first[0] + score_exponent(scale, s.d) > kMostScore;
  const float factor = fabsf(scale) * kLog2e;
  floatx16 o[NB] = {};
  RunningScale ks;
  auto store = [&](int exponent) {
    if (!live) return;
    float* out = dq;
    if (q_parts > 1) out = f.parts + key_parts(s, parts) + part * (static_cast<size_t>(s.b) * s.sq * s.hq * s.d);
#pragma unroll
    for (int n = 0; n < NB; n++) store_columns(out + at, n, half, s.d, o[n], scale, exponent);
  };
  if (__builtin_expect(exact, 0)) {
    tile_barrier();
    const size_t stride = static_cast<size_t>(s.hk) * s.d, of_head = static_cast<size_t>(b) * s.sk * stride + static_cast<size_t>(hk) * s.d;
    const auto* again = args_again<GradArgs>();
    const float *k = again->k, *v = again->v;
    for (int kb = begin; kb < min(end, wave_end); kb++) {
      const size_t from = of_head + static_cast<size_t>(kb) * kBlock * stride;
      const int rows = min(kBlock, keys - kb * kBlock);
      const size_t key = min(lane % 32, rows - 1) * stride;
      const floatx16 x = exact_dots<NB>(k + from + key, q + at, s.d);
      floatx16 ds = exact_dots<NB>(v + from + key, g + at, s.d);
#pragma unroll
      for (int r = 0; r < 16; r++)
        ds[r] = kb * kBlock + result_row(r, half) < seen ? exp2f(fmaf(x[r], scale * kLog2e, -m)) * fmaf(ds[r], inv, -delta) : 0.f;
      exact_outer<NB>(o, k + from, stride, rows, s.d, ds, 0, [](int) { return 1.f; });
    }
    store(0);
    return;
  }
  half8 qh[NB * 2], ql[NB * 2], gh[NB * 2], gl[NB * 2];
  const int eq = row_fragments<NB>(q + at, live, s.d, scale < 0.f ? -1.f : 1.f, 1.f, qh, ql);
  const int eg = row_fragments<NB>(g + at, live, s.d, 1.f, inv, gh, gl);
  tile_barrier();
  auto step = [&](const char* now, char* next, int kb) {
    if (kb + 1 < end) copy_tile<kTile, Waves>(tile + static_cast<size_t>(kb + 1) * kTile, next);
    if (kb < wave_end) {
      const char* t = now + lane * 16;
      const int* tail = reinterpret_cast<const int*>(now + kTile - kTail);
      const int ek = uniform(tail[0]), ev = uniform(tail[1]);
      floatx16 x = {}, dp = {};
#pragma unroll
      for (int n = 0; n < NB * 2; n++)
        x = mfma3(*reinterpret_cast<const half8*>(t + n * 2 * kPart), *reinterpret_cast<const half8*>(t + n * 2 * kPart + kPart),
                  qh[n], ql[n], x);
#pragma unroll
      for (int n = 0; n < NB * 2; n++)
        dp = mfma3(*reinterpret_cast<const half8*>(t + kRowBytes<NB> + n * 2 * kPart),
                   *reinterpret_cast<const half8*>(t + kRowBytes<NB> + n * 2 * kPart + kPart), gh[n], gl[n], dp);
      int behind;
      const int change = ks.take(ek, &behind);
      if (change != 0) {
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
          for (int r = 0; r < 16; r++) o[n][r] = ldexpf(o[n][r], change);
      }
      const float fac = ldexpf(factor, -(eq + ek));
      const float of_dp = power(shift - behind - eg - ev), of_delta = delta * power(shift - behind);
      const bool whole = kb < wave_full;
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const float p = __builtin_amdgcn_exp2f(fmaf(x[r], fac, -m));
        dp[r] = p * fmaf(dp[r], of_dp, -of_delta);
        if (!whole) dp[r] = kb * kBlock + result_row(r, half) < seen ? dp[r] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 2; u++) {
        float d[8];
#pragma unroll
        for (int r = 0; r < 8; r++) d[r] = dp[8 * u + r];
        half8 dh, dl;
        cut_probs(d, &dh, &dl);
        const char* kt = t + 2 * kRowBytes<NB> + u * 2 * kPart;
#pragma unroll
        for (int n = 0; n < NB; n++)
          o[n] = mfma3(*reinterpret_cast<const half8*>(kt + n * 4 * kPart),
                       *reinterpret_cast<const half8*>(kt + n * 4 * kPart + kPart), dh, dl, o[n]);
      }
    }
    tile_barrier();
  };
  for (int kb = begin; kb < end; kb += 2) {
    step(even, odd, kb);
    if (kb + 1 < end) step(odd, even, kb + 1);
  }
  store(-shift - ks.ref);
}

// dk and dv. A workgroup: 128 keys of one key head over its part of the query
// blocks that see any of them, head after head of those that read the key
// head. Two waves share 32 keys: one makes the probabilities and dv, the other
// the gradients' products with the values, and from both ds and dk. So neither
// holds more than one operand and one result (a wave with both leaves a matrix
// core to itself, waiting while it does anything else), at the price of the
// probabilities' way through LDS. Scores are not transposed here: a lane holds
// 16 queries of one key, which is what dv^T += G^T P and dk^T += Q^T dS take.
//
// 16 heads of 128 over 4 key heads and 8192 causal tokens: 1624-1700 us, up to 1015
// TFLOP/s of float16 products, the cores busy 50% of the cycles at 2.0 GHz. Bound
// by the two barriers of a step, at which the pair waits for its probabilities and
// all for the next tile: waves wait 43% of their cycles. (With one wave for both, and four for dq, forward and
// gradients took 4.21 ms instead of 3.65; with 64 keys a workgroup and two of
// them a compute unit, out of step with each other, 3.70 instead of 3.56: the
// query tiles are then copied twice as often.)
//
// The rows of a tile are read before the probabilities' barrier, its columns
// after it. Up to two column groups they have one buffer each, refilled while
// the other is read, so that two workgroups fit a compute unit and
// cover each other's waits. More groups leave room for one workgroup, with two
// buffers of whole tiles.
// Which 128 keys, key head, batch and part of the queries a workgroup takes. The
// first keys, seen by the most queries, come first. With lengths, tiles that are
// no sequence's come last, so that those with work to do are spread evenly over
// the chiplets and take no more rounds than they must: 5 x 12 heads of 80 over
// up to 777 keys, where 240 of 420 tiles had work, took 141 us with the tiles in
// one order for all lengths, and 90 so. Lane l counts the tiles of sequence l, for as many
// sequences as there are lanes.
__device__ inline void key_tile(const Shape& s, const int* lengths, int parts, unsigned block, int* kt, int* part, int* hk,
                                int* b) {
  const unsigned each = static_cast<unsigned>(s.hk) * parts;
  unsigned rest = block % each;
  if (lengths && s.b <= 64) {
    const int lane = threadIdx.x % 64, tiles = (s.sk + 127) / 128;
    const int mine = lane < s.b ? (key_count(s, lengths, lane) + 127) / 128 : 0;
    const unsigned long long every = ~0ull >> (64 - s.b);
    for (int t = 0; t < 2 * tiles; t++) {
      const bool empty = t >= tiles;
      const int at = empty ? t - tiles : t;
      const unsigned long long with = __ballot(mine > at);
      unsigned long long left = empty ? every & ~with : with;
      const unsigned count = __popcll(left) * each;
      if (block >= count) {
        block -= count;
        continue;
      }
      for (unsigned n = block / each; n > 0; n--) left &= left - 1;
      *kt = at;
      *b = __ffsll(left) - 1;
      rest = block % each;
      break;
    }
  } else {
    *kt = block / (each * s.b);
    *b = block / each % s.b;
  }
  *part = rest % parts;
  *hk = rest / parts;
}

template <int NB>
constexpr int kGradRows = 2 * kRowBytes<NB> + kTail;
template <int NB>
constexpr int kGradCols = 2 * kColBytes<NB>;
typedef float4 Probs[4][64];  // of a pair: [registers 4 c .. 4 c + 3][lane]

template <int NB, bool kTwo>
__device__ inline void key_grads(float* __restrict__ dk, float* __restrict__ dv, const float* __restrict__ k,
                                 const float* __restrict__ v, const int* __restrict__ lengths, char* __restrict__ ws,
                                 const Shape& s, float scale, int parts, unsigned block, char* rows_a, char* cols_a,
                                 char* rows_b, char* cols_b, Probs* probs) {
  constexpr int kTile = kQueryTile<NB>, Waves = 8;
  constexpr int kCols = kGradCols<NB>;
  const GradSpace f = grad_space<NB>(ws, s);
  const int group = s.hq / s.hk;
  int kt, part, hk, b;
  key_tile(s, lengths, parts, block, &kt, &part, &hk, &b);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, half = lane / 32;
  const int pair = wave % 4;
  const bool of_keys = wave >= 4;  // makes dk, from ds; the other dv, from p
  const int first = kt * 128 + pair * 32, j = first + lane % 32;
  const int keys = key_count(s, lengths, b), offset = s.sk - s.sq;
  const bool live = j < keys;
  // Query blocks that see a key of the workgroup: those from q_first on, the
  // last first, each of all heads; a part takes every parts-th. Workgroups of
  // other keys start with the same blocks and keep about the same pace, so
  // that a chiplet's cache has what one of them read for the others.
  const int q_first = s.causal ? max(0, kt * 128 - offset) / kBlock : 0;
  const int units = kt * 128 < keys ? max(0, f.q_blocks - q_first) * group : 0;

  const size_t q_head = (static_cast<size_t>(b) * s.hq + static_cast<size_t>(hk) * group) * f.q_blocks;
  // Unit u is query block q_blocks - 1 - u / group of head u % group.
  int back = part / group, of_group = part % group;
  const int back_step = parts / group, head_step = parts % group;
  auto unit_tile = [&](int back, int of_group) {
    return f.q_tiles + (q_head + static_cast<size_t>(of_group) * f.q_blocks + (f.q_blocks - 1 - back)) * kTile;
  };
  auto copy_rows = [&](const char* tile, char* to) {
    copy_tile<2 * kRowBytes<NB>, Waves>(tile, to);
    copy_tile<kTail, Waves>(tile + kTile - kTail, to + 2 * kRowBytes<NB>);
  };
  auto copy_cols = [&](const char* tile, char* to) { copy_tile<kCols, Waves>(tile + 2 * kRowBytes<NB>, to); };
  if (part < units) {
    copy_rows(unit_tile(back, of_group), rows_a);
    copy_cols(unit_tile(back, of_group), cols_a);
  }

  const size_t at = (static_cast<size_t>(b) * s.sk + min(j, s.sk - 1)) * s.hk * s.d + static_cast<size_t>(hk) * s.d;
  half8 fh[NB * 2], fl[NB * 2];  // K for the probabilities (its sign with scale's), V for ds
  const int e = row_fragments<NB>((of_keys ? v : k) + at, live, s.d, !of_keys && scale < 0.f ? -1.f : 1.f, 1.f, fh, fl);
  const int norm = values_norm(f.norms + (static_cast<size_t>(b) * s.hk + hk) * f.k_blocks, (keys + kBlock - 1) / kBlock);
  // Whether all of the head's keys and values and of the group's queries and
  // gradients take float32 products, or some blocks of queries.
  const Ranges of_head = widest_of(f.k_ranges + (static_cast<size_t>(b) * s.hk + hk) * f.k_blocks, (keys + kBlock - 1) / kBlock);
  const Tops of_rows = tops_of(f.q_ranges + q_head, group * f.q_blocks);
  const bool exact = spread(of_head.second) > kSpread || spread(of_rows.first) > kSpread || spread(of_rows.second) > kGradSpread ||
                     of_rows.first[0] + of_head.first[0] + score_exponent(scale, s.d) > kMostScore;
  const float factor = fabsf(scale) * kLog2e;
  floatx16 o[NB] = {};
  RunningScale qs, gs;
  tile_barrier();
  auto step = [&](const char* rows, const char* cols, char* next_rows, char* next_cols, int u) {
    const bool more = u + parts < units;
    const int q0 = (f.q_blocks - 1 - back) * kBlock;
    back += back_step;
    of_group += head_step;
    if (of_group >= group) {
      of_group -= group;
      back++;
    }
    const char* next = unit_tile(back, of_group);
    if (kTwo && more) {
      copy_rows(next, next_rows);
      copy_cols(next, next_cols);
    }
    const char* t = rows + lane * 16 + (of_keys ? kRowBytes<NB> : 0);
    const float* tail = reinterpret_cast<const float*>(rows + 2 * kRowBytes<NB>);
    const int* exponents = reinterpret_cast<const int*>(tail) + 64;
    const int eq = uniform(exponents[0]), eg = uniform(exponents[1]), shift = clamp_power(kScoreShift - uniform(exponents[2]) - norm);
    // Whether any of the block's queries sees any of the wave's keys, and it is
    // not among the uneven ones. (Only where there are some does the step wait for
    // the exponents here.)
    bool any = first < keys && (!s.causal || first <= q0 + kBlock - 1 + offset);
    if (__builtin_expect(of_rows.uneven, 0)) {
      asm volatile("");
      any = any && max(eq, eg) < kUneven / 2;
    }
    // m for the probabilities, delta for ds.
    float4 of_row[4];
#pragma unroll
    for (int c = 0; c < 4; c++) of_row[c] = *reinterpret_cast<const float4*>(tail + (of_keys ? 32 : 0) + 8 * c + 4 * half);
    floatx16 x = {};
    int change = 0, up = 0, q_behind = 0;
    if (any) {
      int g_behind;
      const int g_change = gs.take(eg, &g_behind), q_change = qs.take(shift + eq, &q_behind);
      change = of_keys ? q_change : g_change;
      up = kProbShift - g_behind;  // p carries 2^up
#pragma unroll
      for (int n = 0; n < NB * 2; n++)
        x = mfma3(*reinterpret_cast<const half8*>(t + n * 2 * kPart), *reinterpret_cast<const half8*>(t + n * 2 * kPart + kPart),
                  fh[n], fl[n], x);
      if (!of_keys) {
        const float fac = ldexpf(factor, -(eq + e));
        const bool whole = !s.causal || first + 31 <= q0 + offset;
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const float m4[4] = {of_row[c].x, of_row[c].y, of_row[c].z, of_row[c].w};
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float p = __builtin_amdgcn_exp2f(fmaf(x[4 * c + i], fac, static_cast<float>(up) - m4[i]));
            if (!whole) p = j <= q0 + 8 * c + 4 * half + i + offset ? p : 0.f;
            x[4 * c + i] = p;
          }
          probs[pair][c][lane] = make_float4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
        }
      }
    }
    // The probabilities are in LDS, every wave is done with the rows, and, with
    // one buffer, the columns are there. (With two they are since the step
    // began, and its copies are not waited for.)
    if constexpr (kTwo) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    } else {
      tile_barrier();
      if (more) copy_rows(next, next_rows);
    }
    if (any) {
      if (of_keys) {
        // ds, with what p carries taken off again.
        const int off = shift - q_behind - up;
        const float of_dp = power(off - eg - e), of_delta = power(off);
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const float4 pp = probs[pair][c][lane];
          const float p4[4] = {pp.x, pp.y, pp.z, pp.w}, d4[4] = {of_row[c].x, of_row[c].y, of_row[c].z, of_row[c].w};
#pragma unroll
          for (int i = 0; i < 4; i++) x[4 * c + i] = p4[i] * fmaf(x[4 * c + i], of_dp, -d4[i] * of_delta);
        }
      }
      if (change != 0) {
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
          for (int r = 0; r < 16; r++) o[n][r] = ldexpf(o[n][r], change);
      }
      const char* columns = cols + lane * 16 + (of_keys ? 0 : kColBytes<NB>);
#pragma unroll
      for (int w = 0; w < 2; w++) {
        float p[8];
#pragma unroll
        for (int r = 0; r < 8; r++) p[r] = x[8 * w + r];
        half8 ph, pl;
        cut_probs(p, &ph, &pl);
#pragma unroll
        for (int n = 0; n < NB; n++)
          o[n] = mfma3(*reinterpret_cast<const half8*>(columns + (2 * n + w) * 2 * kPart),
                       *reinterpret_cast<const half8*>(columns + (2 * n + w) * 2 * kPart + kPart), ph, pl, o[n]);
      }
    }
    tile_barrier();
    if (!kTwo && more) copy_cols(next, next_cols);
  };
  if constexpr (kTwo) {
    for (int u = exact ? units : part; u < units; u += 2 * parts) {
      step(rows_a, cols_a, rows_b, cols_b, u);
      if (u + parts < units) step(rows_b, cols_b, rows_a, cols_a, u + parts);
    }
  } else {
    for (int u = exact ? units : part; u < units; u += parts) step(rows_a, cols_a, rows_a, cols_a, u);
  }
  if (exact) gs.ref = -kProbShift;  // sums as they are
  if (exact || of_rows.uneven) {
    // All blocks of queries, or those that are uneven in themselves, by waves
    // that share nothing: both of a pair make the probabilities. Sums keep the
    // scales that they have from the even blocks.
    const auto* again = args_again<GradArgs>();
    const float *q = again->q, *k = again->k, *v = again->v, *g = again->g, *stats = again->stats;
    const size_t q_stride = static_cast<size_t>(s.hq) * s.d;
    for (int u = part; u < units; u += parts) {
      const int block = f.q_blocks - 1 - u / group, h = hk * group + u % group, q0 = block * kBlock, rows = min(kBlock, s.sq - q0);
      const float* tail = reinterpret_cast<const float*>(unit_tile(u / group, u % group) + kTile - kTail);
      const int* exponents = reinterpret_cast<const int*>(tail) + 64;
      const int eq = uniform(exponents[0]), eg = uniform(exponents[1]);
      if (!exact && max(eq, eg) < kUneven / 2) continue;
      if (first >= keys || (s.causal && first > q0 + kBlock - 1 + offset)) continue;
      const size_t q_at = (static_cast<size_t>(b) * s.sq + q0) * q_stride + static_cast<size_t>(h) * s.d;
      // A row's and the key's places, made where they are used.
      auto row = [&] {
        int thread = threadIdx.x;
        asm volatile("" : "+v"(thread));
        return min(thread % 32, rows - 1) * q_stride;
      };
      const float* inv = stats + (static_cast<size_t>(s.b) * s.hq + static_cast<size_t>(b) * s.hq + h) * s.sq + q0;
      int change = 0, behind, shift = 0;
      if (!exact) {
        shift = clamp_power(kScoreShift - uniform(exponents[2]) - norm);
        change = of_keys ? qs.take(shift + (eq < kUneven / 2 ? eq : eq - kUneven), &behind)
                         : gs.take(eg < kUneven / 2 ? eg : eg - kUneven, &behind);
      }
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[n][r] = ldexpf(o[n][r], change);
      floatx16 x = exact_dots<NB>(q + q_at + row(), k + at, s.d);
      __builtin_amdgcn_sched_barrier(0);
      auto seen = [&](int i) { return i < rows && (!s.causal || j <= q0 + i + offset); };
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int i = result_row(r, half);
        x[r] = seen(i) ? exp2f(fmaf(x[r], scale * kLog2e, -tail[i])) : 0.f;
      }
      __builtin_amdgcn_sched_barrier(0);
      if (of_keys) {
        floatx16 ds = exact_dots<NB>(g + q_at + row(), v + at, s.d);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const int i = result_row(r, half);
          ds[r] = seen(i) ? ldexpf(x[r] * fmaf(ds[r], inv[min(i, rows - 1)], -tail[32 + i]), shift) : 0.f;
        }
        exact_outer<NB>(o, q + q_at, q_stride, rows, s.d, ds, qs.ref - shift, [](int) { return 1.f; });
      } else {
        exact_outer<NB>(o, g + q_at, q_stride, rows, s.d, x, gs.ref + kProbShift, [&](int i) { return inv[i]; });
      }
    }
  }
  int thread = threadIdx.x;
  asm volatile("" : "+v"(thread));  // the key's place is made again: held through the uneven blocks it would be spilled
  const int key = first + thread % 32;
  if (key >= s.sk) return;
  const size_t all = static_cast<size_t>(s.b) * s.sk * s.hk * s.d;
  float* out = of_keys ? dk : dv;
  if (parts > 1) out = f.parts + 2 * all * part + (of_keys ? 0 : all);
  // Keys past the length take no gradient (their lanes' sums are not of it).
  if (key >= keys) {
#pragma unroll
    for (int n = 0; n < NB; n++) o[n] = floatx16{};
  }
#pragma unroll
  for (int n = 0; n < NB; n++)
    store_columns(out + (static_cast<size_t>(b) * s.sk + key) * s.hk * s.d + static_cast<size_t>(hk) * s.d, n, thread % 64 / 32, s.d, o[n], of_keys ? scale : 1.f, of_keys ? -qs.ref : -kProbShift - gs.ref);
}

// Sums of parts, in order: element e of two arrays of n in a row.
__device__ inline void sum_parts(float* __restrict__ first, float* __restrict__ second, const float* __restrict__ parts,
                                 size_t n, size_t all, int count) {
  for (size_t e = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; e < all; e += static_cast<size_t>(gridDim.x) * 256) {
    float t = 0.f;
    for (int part = 0; part < count; part++) t += parts[all * part + e];
    if (e < n) first[e] = t;
    else second[e - n] = t;
  }
}

// ── small calls ─────────────────────────────────────────────────────────────
// A token at a time, where reading the keys and values is all the work, and
// calls too small to cut their operands for. 16 query rows of one key head
// (query times the heads that share it) a workgroup; keys and values are read
// as they are, by float32 matrix products. A wave takes 16 keys at a time: S
// (16 keys x 16 rows) = K Q^T, lane l holding key l % 16 and every fourth group
// of 4 columns, and O^T += V^T P with the four terms of a product taken as lane
// l's result rows, 4 (l / 16) + r: P is used where it is. Keys are split over
// workgroups until these fill the chip, and joined by a second launch.
//
// Bound by memory: one token of 32 heads of 128 over 8 key heads and 8 x 8192 keys
// reads 537 MB in 94 us, 5.7 TB/s, and with lengths of half that on the average 268
// MB in 46 us, 5.9 TB/s; the join takes 5. A wave loads its next 16 keys and values
// while it works on the last. Small calls are bound by their few dependent steps: 2
// x 4 heads of 32 over 33 tokens 6 us, 8 x 8 of 64 over 256 causal tokens 18.

// Whether rows are whole vectors of four columns, end within one, or are less
// than one.
enum class Columns { Whole, Odd, Few };

// ND: columns in units of 64.
template <int ND, Columns C>
__device__ inline void token(float* __restrict__ y, const float* __restrict__ q, const float* __restrict__ k,
                             const float* __restrict__ v, float* __restrict__ stats, const int* __restrict__ lengths,
                             char* __restrict__ ws, const Shape& s, float scale, int splits, int units) {
  constexpr int kRow = ND * 64 + 4;  // lanes of unlike rows at unlike banks
  __shared__ __attribute__((aligned(16))) float merged[4][16 * kRow];
  __shared__ float ms[4][16], ls[4][16];
  const int group = s.hq / s.hk, tiles = (s.sq * group + 15) / 16;
  // The workgroup's 16 rows, key head, sequence and part of its keys.
  // The last rows of all heads come first: with `causal` they see the most keys
  // (8 x 16 heads of 64 over 128 tokens 20 us head by head, 15 so). Heads go to the
  // chiplets in turn, so that one has all rows of a head's keys.
  const unsigned heads = static_cast<unsigned>(s.b) * s.hk, at = blockIdx.x / splits;
  int split = blockIdx.x % splits, tile = tiles - 1 - at / heads;
  int hk = at % heads % s.hk, b = at % heads / s.hk;
  unsigned each = 0;
  if (units > 0) {
    const unsigned inner = s.hk * tiles;
    const int unit = blockIdx.x / inner, l = threadIdx.x % 64, mine = l < s.b ? key_count(s, lengths, l) : 0;
    each = keys_a_part(s, mine, splits, units);
    int ends = (mine + each - 1) / each;  // of the parts up to and of sequence l
    for (int d = 1; d < 64; d *= 2) {
      const int before = __shfl_up(ends, d);
      if (l >= d) ends += before;
    }
    b = __popcll(__ballot(l < s.b && ends <= unit));
    if (b == s.b) return;  // there are fewer parts
    split = unit - (b > 0 ? __builtin_amdgcn_readlane(ends, max(b - 1, 0)) : 0);
    tile = blockIdx.x % inner % tiles;
    hk = blockIdx.x % inner / tiles;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int n = lane % 16, quad = lane / 16, first = tile * 16, rows = min(16, s.sq * group - first);
  // Row n of the products: query (first + n) / group, head hk * group + (first + n) % group.
  const int row = first + min(n, rows - 1), i = row / group, h = hk * group + row % group;
  const int keys = key_count(s, lengths, b);
  const int per = units > 0 ? each : ((static_cast<unsigned>(keys) + splits - 1) / splits + 63) / 64 * 64;
  const int begin = split * per;
  const int end = min(visible(s, keys, (first + rows - 1) / group), begin + per);
  const int seen = n < rows ? min(end, visible(s, keys, i)) : 0;
  const float* q_row = q + (static_cast<size_t>(b) * s.sq + i) * s.hq * s.d + static_cast<size_t>(h) * s.d;
  const size_t stride = static_cast<size_t>(s.hk) * s.d;
  const size_t head = static_cast<size_t>(b) * s.sk * stride + static_cast<size_t>(hk) * s.d;
  float4 qv[ND * 4];
#pragma unroll
  for (int t = 0; t < ND * 4; t++) qv[t] = load4(q_row, 16 * t + 4 * quad, s.d);
  const float factor = scale * kLog2e;
  float m = -INFINITY, l = 0.f;
  floatx4 o[ND][4] = {};
  // Columns c .. c + 3 of a row, any of the row's own where they lie past its end
  // (they meet zeros of the query, or are not kept).
  auto columns = [&](const float* row, int c) {
    if constexpr (C == Columns::Few) return make_float4(row[min(c, s.d - 1)], row[min(c + 1, s.d - 1)], row[min(c + 2, s.d - 1)], 0.f);
    else return load4_within(row, c, s.d);
  };
  auto placed = [&](const float4& x, int c) {
    if constexpr (C == Columns::Odd) return turn_to(x, c, s.d);
    else return x;
  };
  // 16 keys and values, loaded while the wave works on the 16 before.
  struct Keys {
    float4 kv[ND * 4], vv[4][ND];
  };
  auto load = [&](Keys& to, int j0) {
    const float* k_row = k + head + min(j0 + n, end - 1) * stride;
#pragma unroll
    for (int t = 0; t < ND * 4; t++) to.kv[t] = columns(k_row, 16 * t + 4 * quad);
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int c = 0; c < ND; c++)
        to.vv[r][c] = columns(v + head + min(j0 + 4 * quad + r, end - 1) * stride, 64 * c + 4 * n);
  };
  auto step = [&](const Keys& now, Keys& next, int j0) {
    load(next, j0 + 64);
    floatx4 x = {};
#pragma unroll
    for (int t = 0; t < ND * 4; t++) {
      const float4 kv = placed(now.kv[t], 16 * t + 4 * quad);
      x = __builtin_amdgcn_mfma_f32_16x16x4f32(kv.x, qv[t].x, x, 0, 0, 0);
      x = __builtin_amdgcn_mfma_f32_16x16x4f32(kv.y, qv[t].y, x, 0, 0, 0);
      x = __builtin_amdgcn_mfma_f32_16x16x4f32(kv.z, qv[t].z, x, 0, 0, 0);
      x = __builtin_amdgcn_mfma_f32_16x16x4f32(kv.w, qv[t].w, x, 0, 0, 0);
    }
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      x[r] = j0 + 4 * quad + r < seen ? x[r] * factor : -INFINITY;
      top = fmaxf(top, x[r]);
    }
    if (__any(top > m + kLazy)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float to = top > m + kLazy ? top : m;
      const float old = to == -INFINITY ? 1.f : exp2f(m - to);
      m = to;
      l *= old;
#pragma unroll
      for (int c = 0; c < ND; c++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[c][e] *= old;
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      x[r] = __builtin_amdgcn_exp2f(x[r] - base);
      l += x[r];
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int c = 0; c < ND; c++) {
        const float4 vv = placed(now.vv[r][c], 64 * c + 4 * n);
        o[c][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv.x, x[r], o[c][0], 0, 0, 0);
        o[c][1] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv.y, x[r], o[c][1], 0, 0, 0);
        o[c][2] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv.z, x[r], o[c][2], 0, 0, 0);
        o[c][3] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv.w, x[r], o[c][3], 0, 0, 0);
      }
  };
  if (begin + wave * 16 < end) {
    Keys even, odd;
    load(even, begin + wave * 16);
    for (int j0 = begin + wave * 16; j0 < end; j0 += 128) {
      step(even, odd, j0);
      if (j0 + 64 < end) step(odd, even, j0 + 64);
    }
  }
  // The four waves' sums, joined in LDS: o[c][e][r] is row n, column 64 c +
  // 4 (4 quad + r) + e.
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (quad == 0) {
    ms[wave][n] = m;
    ls[wave][n] = l;
  }
#pragma unroll
  for (int c = 0; c < ND; c++)
#pragma unroll
    for (int r = 0; r < 4; r++)
      *reinterpret_cast<float4*>(&merged[wave][n * kRow + 64 * c + 4 * (4 * quad + r)]) =
          make_float4(o[c][0][r], o[c][1][r], o[c][2][r], o[c][3][r]);
  __syncthreads();
  const RowParts parts = row_parts(ws, s, splits);
  for (int at = threadIdx.x; at < rows * ND * 64; at += 256) {
    const int row = at / (ND * 64), d = at % (ND * 64);
    float top = fmaxf(fmaxf(ms[0][row], ms[1][row]), fmaxf(ms[2][row], ms[3][row]));
    top = top == -INFINITY ? 0.f : top;
    float sum = 0.f, all = 0.f;
    for (int w = 0; w < 4; w++) {
      const float of = exp2f(ms[w][row] - top);
      sum += of * ls[w][row];
      all += of * merged[w][row * kRow + d];
    }
    const int iq = (first + row) / group, hq = hk * group + (first + row) % group;
    const size_t stat = (static_cast<size_t>(b) * s.hq + hq) * s.sq + iq;
    if (splits > 1) {
      const size_t out = split * parts.rows + stat;
      if (d < s.d) parts.o[out * s.d + d] = all;
      if (d == 0) {
        parts.ml[2 * out] = top;
        parts.ml[2 * out + 1] = sum;
      }
    } else {
      const float inv = inverse_sum(sum);
      if (d < s.d) y[(static_cast<size_t>(b) * s.sq + iq) * s.hq * s.d + static_cast<size_t>(hq) * s.d + d] = all * inv;
      if (d == 0) {
        stats[stat] = top;
        stats[parts.rows + stat] = inv;
      }
    }
  }
}

}  // namespace

// Every launch of a call takes the call's arguments.
#define FG_ARGS                                                                                                  \
  float *y, const float *q, const float *k, const float *v, float *stats, const int *lengths, char *ws, int B,   \
      int Sq, int Sk, int Hq, int Hk, int D, int causal, float scale, int splits, int units, unsigned tiles_lo,    \
      unsigned tiles_hi
#define FG_GRAD_ARGS                                                                                             \
  float *dq, const float *q, const float *k, const float *v, const float *y, const float *g, const float *stats, \
      float *dk, float *dv, const int *lengths, char *ws, int parts, int q_parts, int B, int Sq, int Sk, int Hq, \
      int Hk, int D, int causal, float scale
#define FG_SHAPE \
  Shape { B, Sq, Sk, Hq, Hk, D, causal }

#define FG_ATTENTION(NB)                                                                                         \
  extern "C" __global__ void __launch_bounds__(256) fg_attention_pack_##NB(FG_ARGS) {                            \
    pack_keys<NB>(k, v, lengths, ws, B, Sk, Hk, D);                                                              \
  }                                                                                                              \
  extern "C" __global__ void __launch_bounds__(256, (NB) < 4 ? 6 - (NB) : 2) fg_attention_tiles_##NB(FG_ARGS) {                        \
    forward_tiles<NB>(y, q, stats, lengths, ws, FG_SHAPE, scale, splits);                                        \
  }                                                                                                              \
  extern "C" __global__ void __launch_bounds__(256) fg_attention_grad_pack_##NB(FG_GRAD_ARGS) {                  \
    pack_grad<NB>(q, k, v, y, g, stats, lengths, ws, FG_SHAPE);                                                  \
  }                                                                                                              \
  extern "C" __global__ void __launch_bounds__(64 * kQueryGradWaves<NB>, 2)                                      \
      fg_attention_grad_q_##NB(FG_GRAD_ARGS) {                                                                   \
    __shared__ __attribute__((aligned(1024))) char even[kKeyTile<NB>], odd[kKeyTile<NB>];                        \
    query_grads<NB, kQueryGradWaves<NB>>(dq, q, g, stats, lengths, ws, FG_SHAPE, scale, parts, q_parts,          \
                                         blockIdx.x, even, odd);                                                 \
  }                                                                                                              \
  extern "C" __global__ void __launch_bounds__(512, (NB) < 3 ? 4 : 2) fg_attention_grad_kv_##NB(FG_GRAD_ARGS) {  \
    constexpr bool kTwo = (NB) > 2;                                                                              \
    __shared__ __attribute__((aligned(1024))) char rows_a[kGradRows<NB>], cols_a[kGradCols<NB>];                 \
    __shared__ __attribute__((aligned(1024))) char rows_b[kTwo ? kGradRows<NB> : kPart];                         \
    __shared__ __attribute__((aligned(1024))) char cols_b[kTwo ? kGradCols<NB> : kPart];                         \
    __shared__ Probs probs[4];                                                                                   \
    key_grads<NB, kTwo>(dk, dv, k, v, lengths, ws, FG_SHAPE, scale, parts, blockIdx.x, rows_a, cols_a, rows_b,   \
                        cols_b, probs);                                                                          \
  }                                                                                                              \
  extern "C" __global__ void __launch_bounds__(256) fg_attention_grad_sum_##NB(FG_GRAD_ARGS) {                   \
    const Shape s = FG_SHAPE;                                                                                    \
    const GradSpace f = grad_space<NB>(ws, s);                                                                   \
    const size_t n = static_cast<size_t>(B) * Sk * Hk * D, m = static_cast<size_t>(B) * Sq * Hq * D;             \
    if (parts > 1) sum_parts(dk, dv, f.parts, n, 2 * n, parts);                                                  \
    if (q_parts > 1) sum_parts(dq, dq, f.parts + key_parts(s, parts), m, m, q_parts);                            \
  }

FG_ATTENTION(1)
FG_ATTENTION(2)
FG_ATTENTION(3)
FG_ATTENTION(4)

// Both gradients of a call of few tiles in one launch: the workgroups of dk and
// dv, then those of dq, of whose eight waves the ones that have no part
// in a tile leave at once. In this order the units that take two workgroups have
// one of each kind (with the kinds in turn, 16 heads of 32 over 2048 tokens took
// 229 us with their forward pass instead of 189). Both share the two buffers.
#define FG_ATTENTION_GRADS(NB)                                                                                   \
  extern "C" __global__ void __launch_bounds__(512, (NB) < 2 ? 4 : 2) fg_attention_grads_##NB(FG_GRAD_ARGS) {                   \
    constexpr int kOdd = kGradCols<NB> + 4 * static_cast<int>(sizeof(Probs)), kTile = kKeyTile<NB>;              \
    constexpr int Waves = kQueryGradWaves<NB>;                                                                   \
    __shared__ __attribute__((aligned(1024))) char even[kTile > kGradRows<NB> ? kTile : kGradRows<NB>];          \
    __shared__ __attribute__((aligned(1024))) char odd[kTile > kOdd ? kTile : kOdd];                             \
    const unsigned keys = static_cast<unsigned>(B * Hk) * parts * ((Sk + 127) / 128);                            \
    if (blockIdx.x < keys) {                                                                                     \
      key_grads<NB, false>(dk, dv, k, v, lengths, ws, FG_SHAPE, scale, parts, blockIdx.x, even, odd, even, odd,  \
                           reinterpret_cast<Probs*>(odd + kGradCols<NB>));                                       \
    } else if (threadIdx.x < 64 * Waves) {                                                                       \
      query_grads<NB, Waves>(dq, q, g, stats, lengths, ws, FG_SHAPE, scale, parts, q_parts, blockIdx.x - keys,   \
                             even, odd);                                                                         \
    }                                                                                                            \
  }
FG_ATTENTION_GRADS(1)
FG_ATTENTION_GRADS(2)
FG_ATTENTION_GRADS(3)
FG_ATTENTION_GRADS(4)

#define FG_ATTENTION_TOKEN(ND, NAME, COLUMNS)                                                                    \
  extern "C" __global__ void __launch_bounds__(256, 2) fg_attention_token_##NAME(FG_ARGS) {                      \
    token<ND, Columns::COLUMNS>(y, q, k, v, stats, lengths, ws, FG_SHAPE, scale, splits, units);                   \
  }
FG_ATTENTION_TOKEN(1, 1, Whole)
FG_ATTENTION_TOKEN(2, 2, Whole)
FG_ATTENTION_TOKEN(1, 1_odd, Odd)
FG_ATTENTION_TOKEN(2, 2_odd, Odd)
FG_ATTENTION_TOKEN(1, 1_few, Few)

// The parts begin `tiles` bytes into the workspace (given as two words). W
// columns a thread.
#define FG_ATTENTION_JOIN(W, NAME, ONE_LENGTH)                                                                   \
  extern "C" __global__ void __launch_bounds__(256) fg_attention_join_##NAME(FG_ARGS) {                          \
    join_parts<W, ONE_LENGTH>(y, stats, lengths, ws + (static_cast<size_t>(tiles_hi) << 32 | tiles_lo),          \
                              FG_SHAPE, splits, units);                                                          \
  }
FG_ATTENTION_JOIN(1, 1, false)
FG_ATTENTION_JOIN(4, 4, false)
FG_ATTENTION_JOIN(1, 1_even, true)
FG_ATTENTION_JOIN(4, 4_even, true)
