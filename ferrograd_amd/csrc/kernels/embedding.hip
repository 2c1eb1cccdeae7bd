// Rows of an embedding by token, scaled, and the weight's gradient.
//
//   y_t = s W[id_t],  dW_v = s sum over the tokens t with id_t = v of g_t,
// in an order that the ids and the sizes decide. An id outside of [0, vocab) is
// no token: its row is of zeros, and it has no gradient.
//
// Both are bound by memory: the lookup reads and writes each token's row once,
// the gradient reads each token's row once and writes every row of dW.
//
// Gradient. The tokens are sorted by id, those of an id in their own order,
// while other workgroups of the same launches fill dW with zeros. Then the
// sorted tokens are cut into chunks of one length, however many of them are of
// one id: a group of lanes sums a chunk's rows, writes the sum of an id that
// begins and ends within it to dW, and that of one which goes over its ends to
// the workspace, where a last launch joins it with its other parts. So a padding
// token that is a third of the batch costs no more than any other.
//
// 65536 tokens of 2048 columns, 50001 rows, a third of the tokens one, TB/s of
// what goes past the L2 caches: lookup 138 us (5.2 TB/s; 155 us with a branch
// between a group's loads, which then wait for each other), sort and zeros 66 (6.2;
// the sort alone would take 24), sums 127 (5.1; 174 us with loads that stay in the
// caches), joins 12. What is written twice, the rows that have tokens, is 107 MB
// beside the 1.9 GB that the calls cannot do without.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "vectors.hpp"

namespace {

// A row in slices of G * VEC columns, a slice on G lanes. The last lane of a row
// begins where its vector ends with the row: what it shares with the lane before
// it is the same value again.
template <int VEC, int G>
__device__ inline int column(int slice, int dim) {
  return min((slice * G + static_cast<int>(threadIdx.x) % G) * VEC, dim - VEC);
}

constexpr int kRows = 4;  // tokens that a group of lanes looks up at a time

template <int VEC, int G, bool Stream>
__device__ inline void lookup(float* __restrict__ out, const float* __restrict__ weight, const int* __restrict__ ids,
                              int tokens, int vocab, int dim, int slices, float scale) {
  const unsigned group = (blockIdx.x * 256u + threadIdx.x) / G;
  const int slice = static_cast<int>(group % slices);
  int first = static_cast<int>(group / slices) * kRows;
  const int at = column<VEC, G>(slice, dim);
  auto look_up = [&](auto count) {
    constexpr int N = decltype(count)::value;
    int id[N];
#pragma unroll
    for (int k = 0; k < N; k++) id[k] = ids[first + k];
    Vec<VEC> v[N];
#pragma unroll
    for (int k = 0; k < N; k++)
      v[k] = load<VEC>(weight + static_cast<size_t>(static_cast<unsigned>(id[k]) < static_cast<unsigned>(vocab) ? id[k] : 0) * dim + at);
#pragma unroll
    for (int k = 0; k < N; k++) {
      const bool inside = static_cast<unsigned>(id[k]) < static_cast<unsigned>(vocab);
#pragma unroll
      for (int e = 0; e < VEC; e++) v[k].v[e] = inside ? v[k].v[e] * scale : 0.f;
      store<VEC, Stream>(out + static_cast<size_t>(first + k) * dim + at, v[k]);
    }
  };
  // Whole groups without a branch between their loads, which would wait for each other.
  if (first + kRows <= tokens) {
    look_up(std::integral_constant<int, kRows>());
  } else {
    for (; first < tokens; first++) look_up(std::integral_constant<int, 1>());
  }
}

// ── the tokens in the order of their ids ────────────────────────────────────

// The key that a token is sorted by: its id, or `vocab` where it is none.
__device__ inline unsigned key_of(int id, int vocab) { return min(static_cast<unsigned>(id), static_cast<unsigned>(vocab)); }

// Part `part` of `parts` of dW set to zero, by the workgroups from `first` on.
__device__ inline void fill(float* __restrict__ dw, int vocab, int dim, int first, int part, int parts) {
  typedef float floatx4 __attribute__((ext_vector_type(4)));
  const size_t n = static_cast<size_t>(vocab) * dim, vectors = n / 4, per = (vectors + parts - 1) / parts;
  const size_t end = part + 1 == parts ? vectors : per * (part + 1), step = static_cast<size_t>(gridDim.x - first) * blockDim.x;
  floatx4* to = reinterpret_cast<floatx4*>(dw);
  for (size_t i = per * part + static_cast<size_t>(blockIdx.x - first) * blockDim.x + threadIdx.x; i < end; i += step)
    to[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  if (part == 0 && blockIdx.x == static_cast<unsigned>(first) && threadIdx.x < n % 4) dw[4 * vectors + threadIdx.x] = 0.f;
}

constexpr int kRankThreads = 1024;

// Of up to 12288 tokens: a token's place is the number of tokens before it in
// the order, all of which are looked at. A workgroup ranks 16 tokens against all
// keys, held in LDS: a lane has one of them and every 64th part of the keys, four
// at a time, two and a half vector instructions for 64 pairs. 1000 tokens 3.5 us,
// 5001 7, 16384 would be 31: the four launches below take 25, and more of the host.
constexpr int kRankTokens = 12288, kRanked = 16, kParts = kRankThreads / kRanked;
__device__ inline void rank_tokens(int2* __restrict__ sorted, const int* __restrict__ ids, int tokens, int vocab) {
  __shared__ uint4 keys[kRankTokens / 4];
  __shared__ int places[kParts][kRanked];
  const int part = threadIdx.x / kRanked, own = threadIdx.x % kRanked, t0 = blockIdx.x * kRanked, t = t0 + own;
  unsigned* key = reinterpret_cast<unsigned*>(keys);
  // Past the last token: behind all others.
  // An odd number of vectors a part: the parts that a wave reads are in other banks.
  const int groups = (tokens + 3) / 4, per = (groups + kParts - 1) / kParts | 1;
  for (int i = threadIdx.x; i < 4 * groups; i += kRankThreads) key[i] = i < tokens ? key_of(ids[i], vocab) : 0xffffffffu;
  __syncthreads();
  const unsigned mine = key[min(t, tokens - 1)];
  int before = 0;
#pragma unroll 4
  for (int i = part * per; i < min((part + 1) * per, groups); i++) {
    const uint4 u = keys[i];
    const unsigned below = mine + (4 * i < t0 ? 1u : 0u);  // of the tokens before these also its own key
    before += u.x < below;
    before += u.y < below;
    before += u.z < below;
    before += u.w < below;
  }
  if (part == 0)
    for (int j = 0; j < own; j++) before += key[min(t0 + j, tokens - 1)] == mine;
  places[part][own] = before;
  __syncthreads();
  // A wave sums the parts of 16 tokens, four lanes each.
  if (threadIdx.x >= 64) return;
  before = 0;
#pragma unroll
  for (int k = 0; k < kParts / 4; k++) before += places[4 * k + threadIdx.x / kRanked][own];
  before += __shfl_xor(before, 16);
  before += __shfl_xor(before, 32);
  if (threadIdx.x < kRanked && t < tokens) sorted[before] = make_int2(static_cast<int>(mine), t);
}

// Of more: passes over digits of the key from the lowest on, each keeping the
// order of tokens that it does not tell apart. A workgroup takes `turns` tiles of
// tokens; one launch counts the digits of every workgroup, the next one places the
// tokens. There each reads all counts, so the workgroups are 256 at most: 4 million
// tokens of 50001 ids 45 us for a pass's places, 54 with 512, 129 with one for each
// tile; 30 million 195, 183 with 512, 256 with 1024.
constexpr int kSortThreads = 1024, kWaves = kSortThreads / 64, kItems = 4, kTile = kSortThreads * kItems;
constexpr int kMaxDigits = 1024;

// Token i of a pass: of the first from the ids, later from the last one's order.
__device__ inline int2 token_at(const int2* from, const int* ids, int i, int vocab) {
  return from ? from[i] : make_int2(static_cast<int>(key_of(ids[i], vocab)), i);
}

__device__ inline void count_digits(int* __restrict__ table, const int2* __restrict__ from, const int* __restrict__ ids,
                                    int tokens, int vocab, int shift, int bits, int turns) {
  __shared__ int count[kMaxDigits];
  const int digits = 1 << bits;
  for (int d = threadIdx.x; d < digits; d += kSortThreads) count[d] = 0;
  __syncthreads();
  for (int k = 0; k < kItems * turns; k++) {
    const int i = blockIdx.x * turns * kTile + k * kSortThreads + threadIdx.x;
    if (i < tokens) atomicAdd(&count[(token_at(from, ids, i, vocab).x >> shift) & (digits - 1)], 1);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads) table[blockIdx.x * digits + d] = count[d];
}

__device__ inline void place_tokens(int2* __restrict__ to, const int* __restrict__ table, const int2* __restrict__ from,
                                    const int* __restrict__ ids, int tokens, int vocab, int shift, int bits, int groups, int turns) {
  // Of each wave's digits: how many so far, then how many of the tile's are before them.
  __shared__ int count[kWaves][kMaxDigits];
  __shared__ int base[kMaxDigits], part[kWaves];
  const int digits = 1 << bits, lane = threadIdx.x % 64, wave = threadIdx.x / 64, d = threadIdx.x;
  if (d < digits)
    for (int w = 0; w < kWaves; w++) count[w][d] = 0;
  // Where the digit's tokens of this workgroup begin: after all tokens of lower
  // digits and the earlier workgroups' of this one. One digit a thread.
  int all = 0, earlier = 0;
  if (d < digits)
#pragma unroll 8
    for (int b = 0; b < groups; b++) {
      const int n = table[b * digits + d];
      all += n;
      earlier += b < static_cast<int>(blockIdx.x) ? n : 0;
    }
  int lower = all;
#pragma unroll
  for (int k = 1; k < 64; k *= 2) {
    const int x = __shfl_up(lower, k);
    if (lane >= k) lower += x;
  }
  if (lane == 63) part[wave] = lower;
  __syncthreads();
  lower -= all;
  for (int w = 0; w < wave; w++) lower += part[w];
  lower += earlier;
  if (d < digits) base[d] = lower;
  for (int turn = 0;;) {
    // A wave's tokens in their order, 64 at a time; those of one digit find each
    // other by ballots, and the first of them adds them to the wave's count.
    int2 token[kItems];
    int digit[kItems], place[kItems];
#pragma unroll
    for (int k = 0; k < kItems; k++) {
      const int i = (blockIdx.x * turns + turn) * kTile + (wave * kItems + k) * 64 + lane;
      token[k] = token_at(from, ids, min(i, tokens - 1), vocab);
      digit[k] = i < tokens ? (token[k].x >> shift) & (digits - 1) : -1;
    }
#pragma unroll
    for (int k = 0; k < kItems; k++) {
      unsigned long long same = __ballot(digit[k] >= 0);
      for (int b = 0; b < bits; b++) {
        const bool set = (digit[k] >> b) & 1;
        const unsigned long long ones = __ballot(set);
        same &= set ? ones : ~ones;
      }
      if (digit[k] < 0) same = 1ull << lane;
      const int leader = __ffsll(same) - 1;
      int n = 0;
      if (digit[k] >= 0 && lane == leader) n = atomicAdd(&count[wave][digit[k]], __popcll(same));
      place[k] = __shfl(n, leader) + __popcll(same & ((1ull << lane) - 1));
    }
    __syncthreads();
    if (d < digits) {
      int n = 0;
      for (int w = 0; w < kWaves; w++) {
        const int x = count[w][d];
        count[w][d] = n;
        n += x;
      }
      lower += n;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kItems; k++)
      if (digit[k] >= 0) to[base[digit[k]] + count[wave][digit[k]] + place[k]] = token[k];
    if (++turn == turns) break;
    __syncthreads();
    if (d < digits) {
      for (int w = 0; w < kWaves; w++) count[w][d] = 0;
      base[d] = lower;
    }
    __syncthreads();
  }
}

// ── their rows, summed ──────────────────────────────────────────────────────

constexpr int kBatch = 8;  // rows on their way at a time
// Rows of a float32 sum: those of longer chunks are added up in 64 bits, as the
// chunks are. In float32 throughout, 1024 rows of one id were off by up to 237
// half steps, 4096 by 945.
constexpr int kRun = 64;

// A chunk's parts in the workspace: [chunk][of an id that began before it, of one
// that goes on after it][dim].
template <int VEC, int G, bool Stream>
__device__ inline void sum_chunks(float* __restrict__ dw, const float* __restrict__ g, const int2* __restrict__ sorted,
                                  float* __restrict__ parts, int tokens, int vocab, int dim, int slices, int chunk, int chunks,
                                  float scale) {
  const unsigned group = (blockIdx.x * 256u + threadIdx.x) / G;
  const int slice = static_cast<int>(group % slices), c = static_cast<int>(group / slices);
  if (c >= chunks) return;
  const int at = column<VEC, G>(slice, dim), begin = c * chunk, end = min(begin + chunk, tokens);
  int id = sorted[begin].x;
  if (id >= vocab) return;  // and all behind it
  bool before = begin > 0 && sorted[begin - 1].x == id;
  const int next = end < tokens ? sorted[end].x : vocab;
  Vec<VEC> sum{};
  // Of the id's rows before sum's, a thread's own. In registers they would leave
  // room for four waves a SIMD, not five.
  __shared__ double runs[VEC][256];
  const bool many = chunk > kRun;
  if (many)
#pragma unroll
    for (int e = 0; e < VEC; e++) runs[e][threadIdx.x] = 0.0;
  auto flush = [&](bool after) {
    if (many)
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        sum.v[e] = static_cast<float>(runs[e][threadIdx.x] + sum.v[e]);
        runs[e][threadIdx.x] = 0.0;
      }
    if (before || after) {
      store<VEC>(parts + (static_cast<size_t>(c) * 2 + (before ? 0 : 1)) * dim + at, sum);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; e++) sum.v[e] *= scale;
      store<VEC>(dw + static_cast<size_t>(id) * dim + at, sum);
    }
  };
  for (int i0 = begin; i0 < end; i0 += kBatch) {
    int2 token[kBatch];
    Vec<VEC> v[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; k++) token[k] = sorted[min(i0 + k, end - 1)];
#pragma unroll
    for (int k = 0; k < kBatch; k++) v[k] = load<VEC, Stream>(g + static_cast<size_t>(token[k].y) * dim + at);
    if (many && (i0 - begin) % kRun == 0)
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        runs[e][threadIdx.x] += sum.v[e];
        sum.v[e] = 0.f;
      }
#pragma unroll
    for (int k = 0; k < kBatch; k++) {
      if (i0 + k >= end || token[k].x >= vocab) break;
      if (token[k].x != id) {
        flush(false);
        before = false;
        id = token[k].x;
        sum = v[k];
      } else {
#pragma unroll
        for (int e = 0; e < VEC; e++) sum.v[e] += v[k].v[e];
      }
    }
  }
  flush(next == id);
}

constexpr int kJoinThreads = 256;

// An id that begins in chunk c and goes on: its parts, in 64 bits, those of the
// later chunks shared out to the workgroup's groups of lanes.
template <int VEC, int G>
__device__ inline void join_chunks(float* __restrict__ dw, const int2* __restrict__ sorted, const float* __restrict__ parts,
                                   int tokens, int vocab, int dim, int slices, int chunk, int chunks, float scale) {
  constexpr int kGroups = kJoinThreads / G;
  __shared__ double sums[kGroups][G * VEC];
  const int slice = static_cast<int>(blockIdx.x) % slices, c = static_cast<int>(blockIdx.x) / slices;
  const int begin = c * chunk, end = begin + chunk, id = sorted[end].x;
  if (id >= vocab || sorted[end - 1].x != id || (begin > 0 && sorted[begin].x == id && sorted[begin - 1].x == id)) return;
  // The chunks that begin with it.
  int more = 0;
  for (unsigned long long all = ~0ull; all == ~0ull;) {
    const int d = c + 1 + more + static_cast<int>(threadIdx.x) % 64;
    all = __ballot(d < chunks && sorted[min(d, chunks - 1) * chunk].x == id);
    more += all == ~0ull ? 64 : __ffsll(~all) - 1;
  }
  const int at = column<VEC, G>(slice, dim), group = threadIdx.x / G, lane = threadIdx.x % G;
  double sum[VEC] = {};
  const float* of = parts + static_cast<size_t>(c) * 2 * dim + at;
  if (group == 0) {
    const Vec<VEC> v = load<VEC>(of + dim);
#pragma unroll
    for (int e = 0; e < VEC; e++) sum[e] = v.v[e];
  }
#pragma unroll 8
  for (int k = group; k < more; k += kGroups) {
    const Vec<VEC> v = load<VEC>(of + static_cast<size_t>(k + 1) * 2 * dim);
#pragma unroll
    for (int e = 0; e < VEC; e++) sum[e] += v.v[e];
  }
#pragma unroll
  for (int e = 0; e < VEC; e++) sums[group][lane * VEC + e] = sum[e];
  __syncthreads();
  if (group != 0) return;
  Vec<VEC> total;
#pragma unroll
  for (int e = 0; e < VEC; e++) {
    double t = 0.0;
    for (int k = 0; k < kGroups; k++) t += sums[k][lane * VEC + e];
    total.v[e] = static_cast<float>(t * scale);
  }
  store<VEC>(dw + static_cast<size_t>(id) * dim + at, total);
}

}  // namespace

#define FG_LOOKUP_AS(VEC, G, NAME, STREAM)                                                                             \
  extern "C" __global__ void __launch_bounds__(256) fg_embedding_##NAME(                                               \
      float* out, const float* weight, const int* ids, int tokens, int vocab, int dim, int slices, float scale) {      \
    lookup<VEC, G, STREAM>(out, weight, ids, tokens, vocab, dim, slices, scale);                                       \
  }

// Of the gradient's launches: `sort` workgroups that sort, before those that fill;
// the sorted tokens are at `sorted`, of digits of `bits` bits; `other` is the
// second place of tokens, `table` the counts of digits.
#define FG_GRAD_ARGS                                                                                                    \
  float *dw, const int *ids, const float *g, int2 *sorted, int2 *other, int *table, float *parts, int tokens, int vocab, \
      int dim, int slices, int chunk, int chunks, int sort, int turns, int bits, float scale

#define FG_SUM_AS(VEC, G, NAME, STREAM)                                                                                 \
  extern "C" __global__ void __launch_bounds__(256) fg_embedding_grad_sum_##NAME(FG_GRAD_ARGS) {                        \
    sum_chunks<VEC, G, STREAM>(dw, g, sorted, parts, tokens, vocab, dim, slices, chunk, chunks, scale);                 \
  }

#define FG_EMBEDDING(VEC, G)                                                                                            \
  FG_LOOKUP_AS(VEC, G, VEC##_##G, false)                                                                                \
  FG_LOOKUP_AS(VEC, G, VEC##_##G##_stream, true)                                                                        \
  FG_SUM_AS(VEC, G, VEC##_##G, false)                                                                                   \
  FG_SUM_AS(VEC, G, VEC##_##G##_stream, true)                                                                           \
  extern "C" __global__ void __launch_bounds__(kJoinThreads) fg_embedding_grad_join_##VEC##_##G(FG_GRAD_ARGS) {         \
    join_chunks<VEC, G>(dw, sorted, parts, tokens, vocab, dim, slices, chunk, chunks, scale);                           \
  }

FG_EMBEDDING(1, 8)
FG_EMBEDDING(4, 8)
FG_EMBEDDING(4, 16)
FG_EMBEDDING(4, 32)
FG_EMBEDDING(4, 64)

extern "C" __global__ void __launch_bounds__(kRankThreads) fg_embedding_grad_rank(FG_GRAD_ARGS) {
  if (static_cast<int>(blockIdx.x) < sort) rank_tokens(sorted, ids, tokens, vocab);
  else fill(dw, vocab, dim, sort, 0, 1);
}

// Pass P of `PASSES`: the tokens go from place to place so that the last pass
// leaves them at `sorted`.
#define FG_SORT(P, PASSES)                                                                                              \
  extern "C" __global__ void __launch_bounds__(kSortThreads) fg_embedding_grad_count_##P##_##PASSES(FG_GRAD_ARGS) {     \
    const int2* from = P == 0 ? nullptr : (PASSES - P) % 2 ? other : sorted;                                            \
    if (static_cast<int>(blockIdx.x) < sort) count_digits(table, from, ids, tokens, vocab, P * bits, bits, turns);      \
    else fill(dw, vocab, dim, sort, 2 * P, 2 * PASSES);                                                                 \
  }                                                                                                                     \
  extern "C" __global__ void __launch_bounds__(kSortThreads) fg_embedding_grad_place_##P##_##PASSES(FG_GRAD_ARGS) {     \
    const int2* from = P == 0 ? nullptr : (PASSES - P) % 2 ? other : sorted;                                            \
    if (static_cast<int>(blockIdx.x) < sort)                                                                            \
      place_tokens((PASSES - P) % 2 ? sorted : other, table, from, ids, tokens, vocab, P * bits, bits, sort, turns);    \
    else fill(dw, vocab, dim, sort, 2 * P + 1, 2 * PASSES);                                                             \
  }

FG_SORT(0, 1)
FG_SORT(0, 2)
FG_SORT(1, 2)
FG_SORT(0, 3)
FG_SORT(1, 3)
FG_SORT(2, 3)
FG_SORT(0, 4)
FG_SORT(1, 4)
FG_SORT(2, 4)
FG_SORT(3, 4)
