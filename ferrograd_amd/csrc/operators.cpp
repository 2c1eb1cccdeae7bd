// Graph nodes, gradients and launches of the hand-written kernels.
#include "operators.hpp"

#include <algorithm>
#include <cmath>
#include <cstring>

#include "tensor.hpp"

// The kernels' code objects, compiled for gfx950 from kernels/*.hip when the
// library is built.
#define FG_IMAGE(name)                                     \
  extern "C" const unsigned char fg_image_##name[];        \
  extern "C" const unsigned char fg_image_##name##_end[];
FG_IMAGE(dropout)
FG_IMAGE(norm_rotate)
FG_IMAGE(attention)
FG_IMAGE(embedding)
FG_IMAGE(layer_norm)
FG_IMAGE(token_loss)
FG_IMAGE(clip)

namespace fg {

namespace {

void set_image(RenderedKernel& rk, const unsigned char* begin, const unsigned char* end) {
  rk.image = begin;
  rk.image_size = static_cast<size_t>(end - begin);
}

// Outputs from this size on are written past the caches: they would not stay in
// the Infinity Cache (256 MB) for their reader, and push out what it holds.
constexpr uint64_t kStreamBytes = uint64_t(64) << 20;

int64_t to_bits(double f) {
  int64_t b;
  std::memcpy(&b, &f, 8);
  return b;
}

double from_bits(int64_t b) {
  double f;
  std::memcpy(&f, &b, 8);
  return f;
}

// A call's parameters (its Arg past the output's shape).
std::vector<int64_t> params_of(const UOp& call) {
  const Arg& a = call.arg();
  return std::vector<int64_t>(a.v.begin() + a.b, a.v.end());
}

Shape shape_of(const UOp& call) {
  const Arg& a = call.arg();
  return Shape(a.v.begin(), a.v.begin() + a.b);
}

// A matrix a call reads: as it is, except that a literal is written out first,
// and a tensor with an in-place update not yet realised goes the way it goes in
// every other op.
UOp source(const UOp& u) {
  UOp b = u;
  while (b.op() == Op::Reshape) b = b.src(0);
  return b.op() == Op::Const || b.op() == Op::After ? UOp::contiguous(u) : u;
}

// Whether every element of `u` is the literal 1.
bool is_ones(UOp u) {
  while (u.op() == Op::Reshape || u.op() == Op::Expand) u = u.src(0);
  return u.op() == Op::Const && u.is_const_float(1.0);
}

// A gradient as a call reads it. `y.mul(g).sum(...)`, the way to seed a
// gradient, arrives as g times an expanded 1: the same values without writing
// the product out.
UOp gradient_source(UOp g) {
  while (g.op() == Op::Mul) {
    if (is_ones(g.src(1))) g = g.src(0);
    else if (is_ones(g.src(0))) g = g.src(1);
    else break;
  }
  return source(g);
}

UOp word(uint64_t v, DeviceId d) { return UOp::const_int(static_cast<int32_t>(static_cast<uint32_t>(v)), DType::I32(), d); }

UOp make_call(KernelId id, const Shape& out, const std::vector<UOp>& srcs, const std::vector<int64_t>& params) {
  return UOp::make_new(Op::Kernel, DType::F32(), srcs, Arg::kernel(static_cast<int64_t>(id), out, params));
}

// The device check every operator makes once its arguments are in order.
void need_hip(const Tensor& t, const char* what) {
  FG_CHECK(t.device() == DeviceId::Hip, std::string(what) + ": the " + device_name(t.device()) +
                                            " device has no kernel for it (only hip has)");
}

// A launch of `grid` workgroups. The device counts a launch's threads in 32 bits.
LaunchSpec launch(const std::string& func, uint64_t grid, unsigned block, const char* what, unsigned lds = 0) {
  FG_CHECK(grid >= 1 && grid <= 0xffffffffULL / block,
           std::string(what) + ": " + std::to_string(grid) + " workgroups of " + std::to_string(block) +
               " threads in one launch, which takes 2^32 - 1 threads");
  LaunchSpec l;
  l.func = func;
  l.grid[0] = static_cast<unsigned>(grid);
  l.block[0] = block;
  l.lds_bytes = lds;
  return l;
}

// ── dropout ─────────────────────────────────────────────────────────────────
// params: p's bits.

RenderedKernel render_dropout(const UOp& call) {
  const double p = from_bits(params_of(call)[0]);
  const uint64_t n = numel(shape_of(call));
  RenderedKernel rk;
  rk.kind = "dropout";
  set_image(rk, fg_image_dropout, fg_image_dropout_end);
  const uint64_t threshold = static_cast<uint64_t>(p * 4294967296.0);
  // 4 elements a thread (one block of four random words).
  rk.launches = {launch(4 * n >= kStreamBytes ? "fg_dropout_stream" : "fg_dropout", (n + 511) / 512, 128, "dropout")};
  rk.call_args = {CallArg::slot(0), CallArg::slot(1), CallArg::slot(2), CallArg::slot(3), CallArg::slot(4),
                  CallArg::slot(5), CallArg::i32(static_cast<int32_t>(n & 0xffffffffu)),
                  CallArg::i32(static_cast<int64_t>(n >> 32)), CallArg::i32(static_cast<int32_t>(threshold)),
                  CallArg::f32(static_cast<float>(1.0 / (1.0 - p)))};
  return rk;
}

// Output i (from 1 on) of a call with sources `srcs`: its storage, a source of
// the call besides them. Nodes that are alike are one node, so it carries all
// that tells the call from others on the same sources: without the call's
// parameters two calls that differ in nothing else would write one buffer.
UOp output_storage(KernelId id, int64_t i, const Shape& shape, const std::vector<UOp>& srcs, const std::vector<int64_t>& params) {
  std::vector<int64_t> key{i};
  key.insert(key.end(), params.begin(), params.end());
  return UOp::make_new(Op::KernelBuf, DType::F32(), srcs, Arg::kernel(static_cast<int64_t>(id), shape, key));
}

UOp output_of(const UOp& storage, const UOp& call) {
  return UOp::make_new(Op::KernelOut, storage.dtype(), {storage, call}, Arg::none());
}

// ── norm_rotate ─────────────────────────────────────────────────────────────
// params: tokens, heads, dim, bits of eps, bits of base. Sources: x, weight,
// positions; of the gradient also g and dweight's storage.

// A head in vectors of `vec` of each half on `lanes` lanes
// (kernels/norm_rotate.hip).
struct RowSplit {
  int vec, lanes;
  std::string suffix() const { return "_" + std::to_string(vec) + "_" + std::to_string(lanes); }
};

RowSplit row_split(int64_t dim) {
  const int64_t half = dim / 2;
  RowSplit r{half < 4 ? 1 : 4, 8};
  while (r.lanes * r.vec < half) r.lanes *= 2;
  return r;
}

RenderedKernel render_norm_rotate(const UOp& call, bool grad) {
  const std::vector<int64_t> p = params_of(call);
  const int64_t tokens = p[0], heads = p[1], dim = p[2];
  const double eps = from_bits(p[3]), log2_base = std::log2(from_bits(p[4]));
  const RowSplit r = row_split(dim);
  // Tokens whose angles a workgroup makes at a time: as many as it has threads
  // for, more until its groups of lanes have four rows each, fewer while there
  // are not four workgroups a compute unit.
  const int64_t half = dim / 2, groups = 256 / r.lanes;
  int64_t per = std::max<int64_t>(1, 256 / half);
  while (per * heads < 4 * groups && 2 * per * half <= 1024) per *= 2;
  while (per > 1 && (tokens + per - 1) / per < 1024) per /= 2;
  const int64_t blocks = std::min<int64_t>((tokens + per - 1) / per, grad ? 1024 : 2048);
  RenderedKernel rk;
  set_image(rk, fg_image_norm_rotate, fg_image_norm_rotate_end);
  const float hi = static_cast<float>(log2_base);
  const std::vector<CallArg> tail = {CallArg::i32(tokens), CallArg::i32(heads), CallArg::i32(dim), CallArg::i32(per),
                                     CallArg::f32(static_cast<float>(eps)), CallArg::f32(hi),
                                     CallArg::f32(static_cast<float>(log2_base - hi))};
  const std::string name = r.suffix() + (4 * tokens * heads * dim >= static_cast<int64_t>(kStreamBytes) ? "_stream" : "");
  rk.call_args = {CallArg::slot(0), CallArg::slot(1), CallArg::slot(2), CallArg::slot(3)};
  if (!grad) {
    rk.kind = "norm_rotate";
    rk.launches = {launch("fg_norm_rotate" + name, static_cast<uint64_t>(blocks), 256, "norm_rotate")};
  } else {
    rk.kind = "norm_rotate_grad";
    rk.launches = {launch("fg_norm_rotate_grad" + name, static_cast<uint64_t>(blocks), 256, "norm_rotate"),
                   launch("fg_norm_rotate_weight", static_cast<uint64_t>((dim + 15) / 16), 1024, "norm_rotate")};
    rk.workspace_bytes = static_cast<size_t>(blocks * dim) * 4;
    rk.side_outputs = {5};
    for (CallArg a : {CallArg::slot(4), CallArg::slot(5), CallArg::workspace(), CallArg::i32(blocks)}) rk.call_args.push_back(a);
  }
  rk.call_args.insert(rk.call_args.end(), tail.begin(), tail.end());
  return rk;
}

// ── attention ───────────────────────────────────────────────────────────────
// params: batch, sq, sk, heads, kv_heads, dim, causal, whether there are
// lengths, bits of scale. Sources: q, k, v, [lengths], the stats' storage; of
// the gradient: q, k, v, y, g, stats, [lengths], dk's and dv's storage.

// Units of attention's launches: 32 query rows by 32 keys of every wave of a
// workgroup. A unit's us, measured where workgroups fill the chip (16 heads,
// 2048 queries, 1024 to 4096 keys): two of them a compute unit, or one where
// their tiles leave no room for another. A workgroup with a compute unit to
// itself takes less than each of two do, by these factors.
constexpr double kForwardUnit[] = {1.2, 1.7, 2.3, 3.0}, kKeyUnit[] = {2.7, 3.6, 2.8, 3.3}, kQueryUnit[] = {1.4, 2.3, 3.3, 4.0};
constexpr double kForwardAlone = 0.75, kGradAlone = 0.72;
constexpr int64_t kUnits = 256;   // compute units
constexpr int64_t kRangeBytes = 8;  // of a block of cut operands: its ranges
constexpr double kSumLaunch = 8;  // us of a launch that joins parts, beside its bytes

// One kind of workgroups of a launch: `tiles` of them, each over `units` blocks
// of 32 (with `causal` the longest; the average is half of that), or in parts of
// them, which cost `bytes` each, written and read at 5 TB/s. A workgroup's start
// and end cost as much as some units: `ends_alone` where every one has a compute
// unit to itself, 4 otherwise.
struct Work {
  int64_t tiles, units;
  bool causal;
  double us, alone_us, ends_alone, bytes;
  double joined(int64_t parts) const { return parts > 1 ? 2 * bytes * static_cast<double>(parts) / 5e6 : 0; }
};

// A launch's us with `slots` workgroups on the chip at once and the work cut into
// these parts: as long as its longest workgroup, or as all of them together, of
// which the last end half of one after the others (with `causal` they are
// short). Equal workgroups take whole rounds.
double launch_us(const Work* work, const int64_t* parts, int kinds, int64_t slots) {
  int64_t n = 0;
  for (int i = 0; i < kinds; i++) n += work[i].tiles * parts[i];
  double longest = 0, sum = 0, last = 0;
  for (int i = 0; i < kinds; i++) {
    const Work& w = work[i];
    const double p = static_cast<double>(parts[i]), units = static_cast<double>(w.units) / p, ends = n <= kUnits ? w.ends_alone : 4;
    longest = std::max(longest, (units + ends) * (n <= kUnits || kinds > 1 ? w.alone_us : w.us));
    sum += static_cast<double>(w.tiles) * p * (units * (w.causal ? 0.5 : 1) + ends) * w.us;
    last = w.causal || n <= slots ? 0 : (units + ends) * w.us;
  }
  if (kinds == 1 && !work[0].causal) return static_cast<double>((n + slots - 1) / slots) * longest;
  return std::max(longest, sum / static_cast<double>(slots) + 0.5 * last);
}

struct Split {
  int64_t parts;
  double us;
};

Split count_parts(const Work& work, int64_t slots, double join_us, int64_t most) {
  Split best{1, 0};
  for (int64_t parts = 1; parts <= std::min(work.units, most); parts++) {
    const double us = launch_us(&work, &parts, 1, slots) + (parts > 1 ? work.joined(parts) + join_us : 0);
    if (parts == 1 || us < best.us) best = {parts, us};
  }
  return best;
}

RenderedKernel render_attention(const UOp& call, bool grad) {
  const std::vector<int64_t> p = params_of(call);
  const int64_t batch = p[0], sq = p[1], sk = p[2], heads = p[3], kv_heads = p[4];
  const bool causal = p[6] != 0, lengths = p[7] != 0;
  RenderedKernel rk;
  set_image(rk, fg_image_attention, fg_image_attention_end);
  std::vector<CallArg> tail;
  for (int i = 0; i < 7; i++) tail.push_back(CallArg::i32(p[static_cast<size_t>(i)]));
  tail.push_back(CallArg::f32(static_cast<float>(from_bits(p[8]))));
  const int64_t dim = p[5], nb = (dim + 31) / 32, k_blocks = (sk + 31) / 32;
  const uint64_t all_q = static_cast<uint64_t>(batch * sq * heads * dim), all_k = static_cast<uint64_t>(batch * sk * kv_heads * dim);
  if (!grad) {
    rk.kind = "attention";
    uint64_t tile_bytes = 0;
    // The float32 path: 16 rows a workgroup, and each sequence's keys in parts
    // until there are 1024 workgroups, of at least 256 keys in the longest (four
    // rounds of a workgroup's waves). Where these are more than 512 and sequences
    // have lengths, parts are of one length for all sequences: 8 sequences of up
    // to 8192 keys, 32 heads of 128 over 8, 50 to 62 us instead of 51 to 66 with
    // their joins, 4 of up to 16384, 16 heads of 64 over 4, 18 instead of 21; 2 of
    // up to 3000, 12 heads of 80, 19 instead of 16.
    const int64_t rows = sq * (heads / kv_heads), each = kv_heads * ((rows + 15) / 16), pairs = batch * each;
    int64_t splits = std::max<int64_t>(1, std::min({(1024 + pairs - 1) / pairs, sk / 256, int64_t(64)})), units = 0;
    int64_t blocks, per = ((sk + splits - 1) / splits + 63) / 64 * 64;
    if (lengths && batch > 1 && batch <= 64 && splits > 1 && pairs * splits > 512) {
      units = (512 + each - 1) / each;
      splits = std::min({units, sk / 128, int64_t(64)});
      blocks = std::min(units + batch, splits * batch) * each;
    } else {
      splits = (sk + per - 1) / per;
      blocks = pairs * splits;
    }
    // The other cuts its operands first. It is taken where that and its tiles take
    // less than the float32 workgroups: as long as one of them alone, or as all of
    // them, each a start and rounds of 64 keys. Float32 path against cut operands,
    // us: 8 x 8 heads of 64 over 256 causal tokens 18 and 22, one sequence of 512
    // 16 and 20, 2 x 4 heads of 128 over 500 20 and 32, 16 of 128 over 512 47 and
    // 34, 4 x 50 of 128 over 10 and 99 tokens 29 and 20.
    const bool narrow = dim <= 64;
    const double rounds = static_cast<double>((per + 63) / 64) * (causal && splits == 1 ? 0.75 : 1);
    const double token_us = std::max(narrow ? 4 + 1.5 * rounds : 5 + 2 * rounds,
                                     static_cast<double>(blocks) / static_cast<double>(kUnits) * (narrow ? 1 + 1.2 * rounds : 3 + 2.7 * rounds)) +
                            (splits > 1 ? 5 : 0);
    // Up to four parts are joined in one go; more only until they fill the chip
    // (2 x 8 heads of 64 over 800 causal tokens: 22 us with its join in four
    // parts, 26 in six).
    const int64_t tiles = batch * heads * ((sq + 127) / 128);
    const Work work{tiles, k_blocks, causal, kForwardUnit[nb - 1], kForwardAlone * kForwardUnit[nb - 1], 4, 4.0 * static_cast<double>(all_q)};
    const Split split = count_parts(work, 2 * kUnits, kSumLaunch, std::clamp<int64_t>(2 * kUnits / tiles, 4, 64));
    const double tiles_us = 9 + 16.0 * static_cast<double>(all_k) / 4e6 + split.us;
    if (rows <= 16 || token_us <= tiles_us) {
      rk.launches = {launch(std::string("fg_attention_token_") + (narrow ? "1" : "2") + (dim < 4 ? "_few" : dim % 4 ? "_odd" : ""),
                            static_cast<uint64_t>(blocks), 256, "attention")};
    } else {
      units = 0;
      splits = split.parts;
      const uint64_t key_blocks = static_cast<uint64_t>(batch * kv_heads * k_blocks);
      tile_bytes = key_blocks * static_cast<uint64_t>(nb * 8192 + 1024 + kRangeBytes);
      rk.launches = {launch("fg_attention_pack_" + std::to_string(nb), 2 * key_blocks, 256, "attention"),
                     launch("fg_attention_tiles_" + std::to_string(nb), static_cast<uint64_t>(tiles * splits), 256, "attention")};
    }
    rk.workspace_bytes = std::max<uint64_t>(tile_bytes, 4);
    if (splits > 1) {
      const uint64_t all_rows = static_cast<uint64_t>(batch * heads * sq);
      rk.workspace_bytes = tile_bytes + static_cast<uint64_t>(splits) * (4 * all_q + 8 * all_rows);
      const uint64_t columns = dim < 4 ? 1 : 4;  // a thread's
      rk.launches.push_back(launch("fg_attention_join_" + std::to_string(columns) + (units ? "_even" : ""), (all_rows * ((static_cast<uint64_t>(dim) + columns - 1) / columns) + 255) / 256, 256, "attention"));
    }
    rk.call_args = {CallArg::slot(0), CallArg::slot(1), CallArg::slot(2), CallArg::slot(3), CallArg::slot(lengths ? 5 : 4),
                    lengths ? CallArg::slot(4) : CallArg::null(), CallArg::workspace()};
    for (int64_t x : {splits, units, static_cast<int64_t>(static_cast<int32_t>(tile_bytes & 0xffffffffu)), static_cast<int64_t>(tile_bytes >> 32)})
      tail.push_back(CallArg::i32(x));
    rk.side_outputs = {lengths ? 5 : 4};
  } else {
    rk.kind = "attention_grad";
    const std::string nbs = "_" + std::to_string(nb);
    const int64_t q_blocks = (sq + 31) / 32, group = heads / kv_heads;
    const uint64_t nk = static_cast<uint64_t>(batch * kv_heads * k_blocks), nq = static_cast<uint64_t>(batch * heads * q_blocks);
    const int64_t waves = nb < 4 ? 4 : 8;  // kQueryGradWaves
    const int64_t k_tiles = batch * kv_heads * ((sk + 127) / 128), q_tiles = batch * heads * ((sq + 32 * waves - 1) / (32 * waves));
    // Two workgroups a compute unit where they fit.
    const int64_t k_slots = nb < 3 ? 2 * kUnits : kUnits, q_slots = nb < 4 ? 2 * kUnits : kUnits;
    const double k_us = kKeyUnit[nb - 1], q_us = kQueryUnit[nb - 1], k_alone = (nb < 3 ? kGradAlone : 1) * k_us, q_alone = (nb < 4 ? kGradAlone : 1) * q_us;
    Work work[2] = {{k_tiles, q_blocks * group, causal, k_us, k_alone, 2, 8.0 * static_cast<double>(all_k)},
                    {q_tiles, k_blocks, causal, q_us, q_alone, 2, 4.0 * static_cast<double>(all_q)}};
    const Split k_split = count_parts(work[0], k_slots, kSumLaunch, 16);
    const Split q_split = count_parts(work[1], q_slots, k_split.parts > 1 ? 0 : kSumLaunch, 16);
    int64_t parts = k_split.parts, q_parts = q_split.parts;
    // One launch can have both kinds (two workgroups a compute unit of one column
    // group, one of more), and has them where that takes less than two: their
    // starts, ends and last rounds go together. Two launches against one, us a
    // pass with its forward, causal: 8 x 8 heads of 64 over 256 tokens 78 and 59,
    // 4 x 16 of 32 over 512 96 and 77, 8 of 128 over 1024 141 and 120, 2 x 12 of 64
    // over 900 152 and 115. From twice as many tiles as the chip takes on, no call
    // tried was better so.
    bool together = false;
    const int64_t slots = nb == 1 ? 2 * kUnits : kUnits;
    if (k_tiles + q_tiles <= 2 * slots) {
      if (nb > 1) {
        work[0].us = k_alone;
        work[1].us = q_alone;
      }
      double least = k_split.us + q_split.us;
      for (int64_t both[2] = {1, 1}; both[0] <= std::min<int64_t>(16, work[0].units); both[0]++)
        for (both[1] = 1; both[1] <= std::min<int64_t>(16, work[1].units); both[1]++) {
          // The kind that comes first leaves room for the other's longest.
          if (k_tiles * both[0] + q_tiles * both[1] > slots && 8 * k_tiles * both[0] > 7 * slots) continue;
          const double us = launch_us(work, both, 2, slots) + work[0].joined(both[0]) + work[1].joined(both[1]) +
                            (both[0] > 1 || both[1] > 1 ? kSumLaunch : 0);
          if (us >= least) continue;
          together = true;
          least = us;
          parts = both[0];
          q_parts = both[1];
        }
    }
    const uint64_t summed = std::max(parts > 1 ? 2 * all_k : 0, q_parts > 1 ? all_q : 0);
    rk.workspace_bytes = nk * static_cast<uint64_t>(nb * 12288 + 1024 + kRangeBytes) + nq * static_cast<uint64_t>(nb * 16384 + 1024 + kRangeBytes) +
                         (nk + 3) / 4 * 16 + (parts > 1 ? 8 * all_k * static_cast<uint64_t>(parts) : 0) +
                         (q_parts > 1 ? 4 * all_q * static_cast<uint64_t>(q_parts) : 0);
    rk.launches = {launch("fg_attention_grad_pack" + nbs, 2 * (nk + nq), 256, "attention")};
    if (together) {
      rk.launches.push_back(launch("fg_attention_grads" + nbs, static_cast<uint64_t>(k_tiles * parts + q_tiles * q_parts), 512, "attention"));
    } else {
      rk.launches.push_back(launch("fg_attention_grad_kv" + nbs, static_cast<uint64_t>(k_tiles * parts), 512, "attention"));
      rk.launches.push_back(launch("fg_attention_grad_q" + nbs, static_cast<uint64_t>(q_tiles * q_parts), static_cast<unsigned>(64 * waves), "attention"));
    }
    if (summed) rk.launches.push_back(launch("fg_attention_grad_sum" + nbs, std::min<uint64_t>((summed + 255) / 256, 8192), 256, "attention"));
    const int dk = lengths ? 8 : 7;
    for (int i = 0; i < 7; i++) rk.call_args.push_back(CallArg::slot(i));
    rk.call_args.push_back(CallArg::slot(dk));
    rk.call_args.push_back(CallArg::slot(dk + 1));
    rk.call_args.push_back(lengths ? CallArg::slot(7) : CallArg::null());
    rk.call_args.push_back(CallArg::workspace());
    rk.call_args.push_back(CallArg::i32(parts));
    rk.call_args.push_back(CallArg::i32(q_parts));
    rk.side_outputs = {dk, dk + 1};
  }
  rk.call_args.insert(rk.call_args.end(), tail.begin(), tail.end());
  return rk;
}

// ── embedding ───────────────────────────────────────────────────────────────
// params: tokens, vocab, dim, bits of scale. Sources: weight, ids; of the
// gradient ids, g.

// Rows in slices of `lanes` times `vec` columns.
struct ColumnSplit {
  int64_t vec, lanes, slices;
  std::string suffix() const { return "_" + std::to_string(vec) + "_" + std::to_string(lanes); }
};

ColumnSplit column_split(int64_t dim) {
  ColumnSplit r{dim < 4 ? 1 : 4, 8, 1};
  while (r.lanes < 64 && r.lanes * r.vec < dim) r.lanes *= 2;
  r.slices = (dim + r.lanes * r.vec - 1) / (r.lanes * r.vec);
  return r;
}

constexpr int64_t kSortTile = 4096, kSortGroups = 256, kSortDigitBits = 10, kRankTokens = 12288;  // kernels/embedding.hip

RenderedKernel render_embedding(const UOp& call, bool grad) {
  const std::vector<int64_t> p = params_of(call);
  const int64_t tokens = p[0], vocab = p[1], dim = p[2];
  const ColumnSplit split = column_split(dim);
  const float scale = static_cast<float>(from_bits(p[3]));
  RenderedKernel rk;
  set_image(rk, fg_image_embedding, fg_image_embedding_end);
  for (int i = 0; i < 3; i++) rk.call_args.push_back(CallArg::slot(i));
  if (!grad) {
    rk.kind = "embedding";
    const uint64_t groups = static_cast<uint64_t>((tokens + 3) / 4 * split.slices);  // of four tokens each
    rk.launches = {launch("fg_embedding" + split.suffix() + (4 * tokens * dim >= static_cast<int64_t>(kStreamBytes) ? "_stream" : ""),
                          (groups * static_cast<uint64_t>(split.lanes) + 255) / 256, 256, "embedding")};
    for (int64_t x : {tokens, vocab, dim, split.slices}) rk.call_args.push_back(CallArg::i32(x));
    rk.call_args.push_back(CallArg::f32(scale));
    return rk;
  }
  rk.kind = "embedding_grad";
  // Chunks of 32 sorted tokens, shorter while they are too few to fill the chip
  // (up to 2048 of them: the joining launch has a workgroup for each), longer
  // where one id could be in more than 256 for each group of lanes that joins
  // them. Sums and joins: 1000 tokens of 4 columns 9 + 4 us in chunks of 32, 4 + 4
  // in 8; 65536 of 4 columns 5 + 17 in 8, 11 + 7 in 32, 17 + 5 in 64; 65536 of 2048
  // columns 174 + 18 in 32, 174 + 12 in 64.
  int64_t chunk = 32;
  while (chunk > 8 && tokens / chunk < 1024 && tokens / chunk * split.slices * split.lanes < 2048 * 64) chunk /= 2;
  while (tokens / chunk > 256 * (256 / split.lanes)) chunk *= 2;
  const int64_t chunks = (tokens + chunk - 1) / chunk;
  const uint64_t pairs = static_cast<uint64_t>(tokens + tokens % 2) * 8;
  const bool rank = tokens <= kRankTokens;
  int64_t key_bits = 1;
  while (vocab >> key_bits) key_bits++;
  const int64_t passes = rank ? 0 : (key_bits + kSortDigitBits - 1) / kSortDigitBits;
  const int64_t bits = rank ? 0 : (key_bits + passes - 1) / passes;
  const int64_t tiles = (tokens + kSortTile - 1) / kSortTile, turns = (tiles + kSortGroups - 1) / kSortGroups;
  const int64_t sort = rank ? (tokens + 15) / 16 : (tiles + turns - 1) / turns;
  const uint64_t table = rank ? 0 : static_cast<uint64_t>(sort << bits) * 4;
  const uint64_t table_at = pairs + (rank ? 0 : pairs), parts_at = table_at + (table + 15) / 16 * 16;
  rk.workspace_bytes = parts_at + (chunks > 1 ? static_cast<uint64_t>(chunks * 2 * dim) * 4 : 0);
  // Workgroups that fill, four vectors a thread or more.
  const int64_t fill = std::clamp<int64_t>(vocab * dim / 16384 / std::max<int64_t>(1, 2 * passes), 1, 512);
  const uint64_t both = static_cast<uint64_t>(sort + fill);
  if (rank) rk.launches.push_back(launch("fg_embedding_grad_rank", both, 1024, "embedding"));
  for (int64_t i = 0; i < passes; i++)
    for (const char* step : {"count", "place"})
      rk.launches.push_back(launch(std::string("fg_embedding_grad_") + step + "_" + std::to_string(i) + "_" + std::to_string(passes), both, 1024, "embedding"));
  rk.launches.push_back(launch("fg_embedding_grad_sum" + split.suffix() + (4 * tokens * dim >= static_cast<int64_t>(kStreamBytes) ? "_stream" : ""),
                               (static_cast<uint64_t>(chunks * split.slices * split.lanes) + 255) / 256, 256, "embedding"));
  if (chunks > 1)
    rk.launches.push_back(launch("fg_embedding_grad_join" + split.suffix(), static_cast<uint64_t>((chunks - 1) * split.slices), 256, "embedding"));
  for (uint64_t at : {uint64_t(0), pairs, table_at, parts_at}) rk.call_args.push_back(CallArg::workspace(at));
  for (int64_t x : {tokens, vocab, dim, split.slices, chunk, chunks, sort, turns, bits}) rk.call_args.push_back(CallArg::i32(x));
  rk.call_args.push_back(CallArg::f32(scale));
  return rk;
}

// ── layer_norm ──────────────────────────────────────────────────────────────
// params: rows, dim, whether there is a bias, bits of eps. Sources: x, weight,
// [bias]; of the gradient x, weight, g, dweight's and [dbias's] storage.

// A row on `lanes` lanes, up to `vectors` vectors of four each
// (kernels/layer_norm.hip).
struct RegisterSplit {
  int64_t lanes, vectors;
};
constexpr RegisterSplit kLayerNormSplits[] = {{8, 1},  {16, 1},  {32, 1},  {64, 1},  {64, 2},
                                               {64, 4}, {256, 2}, {256, 4}, {512, 4}, {1024, 4}, {1024, 8}};

RenderedKernel render_layer_norm(const UOp& call, bool grad) {
  const std::vector<int64_t> p = params_of(call);
  const int64_t rows = p[0], dim = p[1];
  const bool bias = p[2] != 0;
  RenderedKernel rk;
  set_image(rk, fg_image_layer_norm, fg_image_layer_norm_end);
  const RegisterSplit* split = nullptr;
  for (const RegisterSplit& s : kLayerNormSplits)
    if (!split && 4 * s.lanes * s.vectors >= dim) split = &s;
  const std::string name = !split ? "_long" : "_" + std::to_string(split->lanes) + "_" + std::to_string(split->vectors) +
                                                  (dim % 4 ? "_odd" : "") +
                                                  (4 * rows * dim >= static_cast<int64_t>(kStreamBytes) ? "_stream" : "");
  const int64_t threads = !split ? 1024 : std::max<int64_t>(256, split->lanes), groups = split ? threads / split->lanes : 1;
  const int64_t turns = (rows + groups - 1) / groups;  // workgroups, if each had its rows at once
  for (int i = 0; i < 3; i++) rk.call_args.push_back(CallArg::slot(i));
  if (!grad) {
    rk.kind = "layer_norm";
    rk.launches = {launch("fg_layer_norm" + name, static_cast<uint64_t>(std::min<int64_t>(turns, 8 * kUnits * 256 / threads)),
                          static_cast<unsigned>(threads), "layer_norm")};
    rk.call_args.push_back(bias ? CallArg::slot(3) : CallArg::null());
  } else {
    rk.kind = "layer_norm_grad";
    // Workgroups that fit the chip together, so that each adds up what it can
    // before its sums go to memory.
    int64_t blocks = std::min<int64_t>(turns, 4 * kUnits * 256 / threads);
    rk.launches = {launch("fg_layer_norm_grad" + name, static_cast<uint64_t>(blocks), static_cast<unsigned>(threads), "layer_norm")};
    const bool sums = split && split->vectors < 8;
    if (!sums) {
      blocks = std::min<int64_t>(rows, 32);
      rk.launches.push_back(launch("fg_layer_norm_grad_long_sums", static_cast<uint64_t>((dim + 255) / 256 * blocks), 256, "layer_norm"));
    }
    rk.launches.push_back(launch("fg_layer_norm_weight", static_cast<uint64_t>((2 * dim + 31) / 32), 1024, "layer_norm"));
    const uint64_t stats_at = static_cast<uint64_t>(blocks * 2 * dim) * 4;
    rk.workspace_bytes = stats_at + (sums ? 0 : static_cast<uint64_t>(rows) * 8);
    rk.side_outputs = {4};
    if (bias) rk.side_outputs.push_back(5);
    for (CallArg a : {CallArg::slot(3), CallArg::slot(4), bias ? CallArg::slot(5) : CallArg::null(), CallArg::workspace(),
                      CallArg::workspace(stats_at), CallArg::i32(blocks)})
      rk.call_args.push_back(a);
  }
  rk.call_args.push_back(CallArg::i32(rows));
  rk.call_args.push_back(CallArg::i32(dim));
  rk.call_args.push_back(CallArg::f32(static_cast<float>(from_bits(p[3]))));
  return rk;
}

// ── token_cross_entropy ─────────────────────────────────────────────────────
// params: rows, classes. Sources: logits, labels. Of the gradient also whether it
// makes the loss; sources: logits, labels, and the loss's storage, or else g.

// A row on `lanes` lanes, up to `vectors` vectors of four each
// (kernels/token_loss.hip).
constexpr RegisterSplit kTokenLossSplits[] = {{8, 1},   {16, 1},  {32, 1},  {64, 1},  {64, 2},   {64, 4},
                                               {256, 2}, {256, 4}, {256, 8}, {512, 8}, {1024, 8}, {1024, 16}};

constexpr uint64_t kLossCounts = 16;  // workgroups that count the valid labels

RenderedKernel render_token_loss(const UOp& call, bool grad) {
  const std::vector<int64_t> p = params_of(call);
  const int64_t rows = p[0], classes = p[1];
  const bool joint = grad && p[2] != 0;
  RenderedKernel rk;
  set_image(rk, fg_image_token_loss, fg_image_token_loss_end);
  const RegisterSplit* split = nullptr;
  // Long rows of broken vectors begin on the cache line that their first one is in.
  for (const RegisterSplit& s : kTokenLossSplits)
    if (!split && 4 * s.lanes * s.vectors - (s.lanes * s.vectors >= 2048 && classes % 4 ? 31 : 0) >= classes) split = &s;
  std::string name = !split ? "_long" : "_" + std::to_string(split->lanes) + "_" + std::to_string(split->vectors) + (classes % 4 ? "_odd" : "");
  if (split && grad && 4 * rows * classes >= static_cast<int64_t>(kStreamBytes)) name += "_stream";
  const int64_t threads = !split ? 1024 : std::max<int64_t>(256, split->lanes), groups = split ? threads / split->lanes : 1;
  // A workgroup for each long row, so that those of ignored rows leave theirs to
  // others: 4096 rows of 16000, three tenths ignored, 79 us instead of 88 in as
  // many workgroups as the chip has room for, 8192 of 4000 41 instead of 48. One
  // alone for short rows that it goes through in 8 turns, as it then needs no other
  // launch.
  const int64_t turns = (rows + groups - 1) / groups;
  const int64_t blocks = groups == 1 ? std::min<int64_t>(turns, 1 << 20) : turns <= 8 ? 1 : std::min<int64_t>(turns, 8 * kUnits);
  const int64_t parts = groups == 1 ? rows : blocks;  // of the loss
  for (int i = 0; i < 3; i++) rk.call_args.push_back(CallArg::slot(i));
  if (!grad) {
    rk.kind = "token_loss";
    rk.launches = {launch("fg_token_loss" + name, static_cast<uint64_t>(blocks), static_cast<unsigned>(threads), "token_cross_entropy")};
    if (blocks > 1) rk.launches.push_back(launch("fg_token_loss_mean", 1, 1024, "token_cross_entropy"));
    rk.workspace_bytes = static_cast<uint64_t>(parts) * 8;
    for (CallArg a : {CallArg::workspace(), CallArg::workspace(static_cast<uint64_t>(parts) * 4), CallArg::i32(parts)})
      rk.call_args.push_back(a);
  } else {
    rk.kind = "token_loss_grad";
    // The valid labels are counted by each workgroup, or once (3 us) where they are
    // many.
    const bool count = rows > 2048;
    if (count) rk.launches.push_back(launch("fg_token_loss_grad_count", kLossCounts, 1024, "token_cross_entropy"));
    rk.launches.push_back(launch("fg_token_loss_grad" + name, static_cast<uint64_t>(blocks), static_cast<unsigned>(threads), "token_cross_entropy"));
    if (joint && blocks > 1) rk.launches.push_back(launch("fg_token_loss_grad_mean", 1, 1024, "token_cross_entropy"));
    rk.workspace_bytes = 4 * kLossCounts + static_cast<uint64_t>(parts) * 8;
    rk.call_args.push_back(joint ? CallArg::null() : CallArg::slot(3));
    rk.call_args.push_back(joint ? CallArg::slot(3) : CallArg::null());
    rk.call_args.push_back(joint ? CallArg::workspace(4 * kLossCounts) : CallArg::null());
    rk.call_args.push_back(joint ? CallArg::workspace(4 * kLossCounts + static_cast<uint64_t>(parts) * 4) : CallArg::null());
    rk.call_args.push_back(CallArg::i32(parts));
    rk.call_args.push_back(count ? CallArg::workspace() : CallArg::null());
    if (joint) rk.side_outputs = {3};
  }
  rk.call_args.push_back(CallArg::i32(rows));
  rk.call_args.push_back(CallArg::i32(classes));
  return rk;
}

// ── clip_norm ───────────────────────────────────────────────────────────────
// Square sums' params: workgroups, whether other sums are added, then the
// tensors' sizes; sources: the tensors, [the other sums]. Their result is
// as many numbers of 64 bits, two elements each. Clipping's params: bits of
// max_norm, workgroups of the sums, whether it writes the norm, then the sizes;
// sources: the tensors, the sums, the storage of its outputs after the first,
// [of the norm].

constexpr size_t kClipTensors = 64;  // of a launch (kernels/clip.hip)
constexpr int64_t kClipChunk = 4096;
// Workgroups of a pass over the tensors: enough to fill the chip, each with some
// chunks where there are many.
constexpr int64_t kClipBlocks = 2048;

int64_t clip_chunks(const std::vector<int64_t>& p, size_t first) {
  int64_t chunks = 0;
  for (size_t i = first; i < p.size(); i++) chunks += (p[i] + kClipChunk - 1) / kClipChunk;
  return chunks;
}

// The tensors that a launch has arguments for.
size_t clip_places(size_t count) { return count <= 16 ? 16 : kClipTensors; }

// Addresses and sizes of the tensors, from slot 1 on.
std::vector<CallArg> clip_args(const std::vector<int64_t>& p, size_t first) {
  const size_t count = p.size() - first, places = clip_places(count);
  std::vector<CallArg> a;
  for (size_t i = 0; i < places; i++) a.push_back(i < count ? CallArg::slot(static_cast<int32_t>(i) + 1) : CallArg::null());
  for (size_t i = 0; i < places; i++) a.push_back(CallArg::bits64(i < count ? p[first + i] : 0));
  return a;
}

RenderedKernel render_square_sums(const UOp& call) {
  const std::vector<int64_t> p = params_of(call);
  const int32_t count = static_cast<int32_t>(p.size() - 2);
  RenderedKernel rk;
  set_image(rk, fg_image_clip, fg_image_clip_end);
  rk.kind = "square_sums";
  rk.launches = {launch("fg_square_sums_" + std::to_string(clip_places(p.size() - 2)), static_cast<uint64_t>(p[0]), 256, "clip_norm")};
  rk.call_args = clip_args(p, 2);
  rk.call_args.push_back(CallArg::slot(0));
  rk.call_args.push_back(p[1] ? CallArg::slot(count + 1) : CallArg::null());
  rk.call_args.push_back(CallArg::i32(count));
  return rk;
}

RenderedKernel render_norm_of_sums(const UOp& call) {
  RenderedKernel rk;
  set_image(rk, fg_image_clip, fg_image_clip_end);
  rk.kind = "norm_of_sums";
  rk.launches = {launch("fg_norm_of_sums", 1, 256, "global_norm")};
  rk.call_args = {CallArg::slot(0), CallArg::slot(1), CallArg::i32(params_of(call)[0])};
  return rk;
}

RenderedKernel render_clip(const UOp& call) {
  const std::vector<int64_t> p = params_of(call);
  const bool norm = p[2] != 0;
  const int32_t count = static_cast<int32_t>(p.size() - 3);
  RenderedKernel rk;
  set_image(rk, fg_image_clip, fg_image_clip_end);
  rk.kind = "clip";
  const int64_t chunks = clip_chunks(p, 3);
  rk.launches = {launch("fg_clip_" + std::to_string(clip_places(p.size() - 3)) +
                            (4 * kClipChunk * chunks >= static_cast<int64_t>(kStreamBytes) ? "_stream" : ""),
                        static_cast<uint64_t>(std::min(chunks, kClipBlocks)), 256, "clip_norm")};
  rk.call_args = clip_args(p, 3);
  // Slots: the first output, the tensors, the sums, the further outputs, the norm.
  for (int32_t i = 0; i < static_cast<int32_t>(clip_places(p.size() - 3)); i++)
    rk.call_args.push_back(i >= count ? CallArg::null() : CallArg::slot(i ? count + 1 + i : 0));
  for (int32_t i = 1; i < count + norm; i++) rk.side_outputs.push_back(count + 1 + i);
  rk.call_args.push_back(CallArg::slot(count + 1));
  rk.call_args.push_back(norm ? CallArg::slot(2 * count + 1) : CallArg::null());
  rk.call_args.push_back(CallArg::bits64(p[0]));
  rk.call_args.push_back(CallArg::i32(p[1]));
  rk.call_args.push_back(CallArg::i32(count));
  return rk;
}

// The tensors of a clip as their calls read them.
std::vector<UOp> clip_sources(const std::vector<Tensor>& tensors, const char* what) {
  const std::string name = what;
  FG_CHECK(!tensors.empty(), name + ": there must be at least one tensor");
  std::vector<UOp> out;
  uint64_t chunks = 0;
  for (size_t i = 0; i < tensors.size(); i++) {
    const Tensor& t = tensors[i];
    FG_CHECK(t.dtype() == DType::F32(), name + ": tensor " + std::to_string(i) + " must be f32");
    FG_CHECK(t.numel() > 0, name + ": tensor " + std::to_string(i) + " is empty");
    FG_CHECK(t.device() == tensors[0].device(), name + ": all tensors must be on the same device");
    chunks += (t.numel() + kClipChunk - 1) / kClipChunk;
    out.push_back(source(t.uop()));
  }
  // The kernels count chunks in 32 bits, some workgroups' past the last.
  FG_CHECK(chunks <= (1u << 30), name + ": more than 2^42 elements");
  need_hip(tensors[0], what);
  return out;
}

// The sums of squares of the tensors' chunks, of as many workgroups as `blocks`
// says: kClipTensors tensors a call.
UOp square_sums(const std::vector<UOp>& srcs, int64_t* blocks) {
  int64_t chunks = 0;
  for (const UOp& u : srcs) chunks += (static_cast<int64_t>(numel(u.shape())) + kClipChunk - 1) / kClipChunk;
  *blocks = std::min(chunks, kClipBlocks);
  UOp sums;
  for (size_t first = 0; first < srcs.size(); first += kClipTensors) {
    std::vector<UOp> part(srcs.begin() + static_cast<std::ptrdiff_t>(first),
                          srcs.begin() + static_cast<std::ptrdiff_t>(std::min(srcs.size(), first + kClipTensors)));
    std::vector<int64_t> params{*blocks, first ? 1 : 0};
    for (const UOp& u : part) params.push_back(static_cast<int64_t>(numel(u.shape())));
    if (first) part.push_back(sums);
    sums = make_call(KernelId::SquareSums, Shape{2 * static_cast<size_t>(*blocks)}, part, params);
  }
  return sums;
}

void check_matrix(const Tensor& t, const char* what) {
  FG_CHECK(t.dtype() == DType::F32(), std::string(what) + " must be f32");
  FG_CHECK(t.ndim() == 2, std::string(what) + " must be 2D (one row per token), got shape " + shape_str(t.shape()));
  FG_CHECK(t.numel() > 0, std::string(what) + " is empty");
}

}  // namespace

Tensor Tensor::norm_rotate(const Tensor& weight, const Tensor& positions, size_t heads, double eps, double base) const {
  check_matrix(*this, "norm_rotate: the input");
  FG_CHECK(device() == weight.device() && device() == positions.device(), "norm_rotate: all tensors must be on the same device");
  const Shape s = shape();
  FG_CHECK(heads >= 1 && s[1] % heads == 0,
           "norm_rotate: " + std::to_string(s[1]) + " columns do not split into " + std::to_string(heads) + " heads");
  const size_t dim = s[1] / heads;
  FG_CHECK(dim % 2 == 0 && dim <= 512, "norm_rotate: the head size must be even and at most 512, got " + std::to_string(dim));
  FG_CHECK(weight.dtype() == DType::F32() && weight.shape() == Shape{dim},
           "norm_rotate: the weight must be f32 of shape " + shape_str(Shape{dim}) + ", got " + shape_str(weight.shape()));
  FG_CHECK(positions.dtype() == DType::I32() && positions.shape() == Shape{s[0]},
           "norm_rotate: the positions must be i32 of shape " + shape_str(Shape{s[0]}) + ", got " + shape_str(positions.shape()));
  // As float32, which the kernels add: infinity would give 0, and 0 NaN for a row of zeros.
  FG_CHECK(eps >= 0 && std::isfinite(static_cast<float>(eps)) && (eps == 0 || static_cast<float>(eps) > 0),
           "norm_rotate: eps must be finite and not negative, and not 0 in float32 unless it is 0");
  FG_CHECK(base > 0 && std::isfinite(base), "norm_rotate: base must be finite and positive");
  // The kernels count rows in 32 bits, some workgroups' rows past the last.
  FG_CHECK(s[0] * heads <= 0x7fffffffu - 1024, "norm_rotate: more than 2^31 - 1025 heads of tokens");
  need_hip(*this, "norm_rotate");
  return from_uop(make_call(KernelId::NormRotate, s, {source(uop()), source(weight.uop()), source(positions.uop())},
                            {static_cast<int64_t>(s[0]), static_cast<int64_t>(heads), static_cast<int64_t>(dim),
                             to_bits(eps), to_bits(base)}),
                  requires_grad() || weight.requires_grad());
}

Tensor Tensor::attention(const Tensor& k, const Tensor& v, const Tensor* lengths, size_t batch, size_t heads,
                         size_t kv_heads, bool causal, double scale) const {
  check_matrix(*this, "attention: q");
  check_matrix(k, "attention: k");
  check_matrix(v, "attention: v");
  FG_CHECK(device() == k.device() && device() == v.device() && (!lengths || device() == lengths->device()),
           "attention: all tensors must be on the same device");
  const Shape qs = shape(), ks = k.shape();
  FG_CHECK(batch >= 1 && qs[0] % batch == 0 && ks[0] % batch == 0,
           "attention: " + std::to_string(qs[0]) + " query rows and " + std::to_string(ks[0]) +
               " key rows do not split into a batch of " + std::to_string(batch));
  FG_CHECK(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0,
           "attention: " + std::to_string(heads) + " heads do not share " + std::to_string(kv_heads) + " key heads evenly");
  FG_CHECK(qs[1] % heads == 0, "attention: " + std::to_string(qs[1]) + " columns do not split into " + std::to_string(heads) + " heads");
  const size_t dim = qs[1] / heads;
  FG_CHECK(dim <= 128, "attention: the head size must be at most 128, got " + std::to_string(dim));
  FG_CHECK(ks[1] == kv_heads * dim, "attention: k must have " + std::to_string(kv_heads) + " heads of " + std::to_string(dim) +
                                        ", got " + std::to_string(ks[1]) + " columns");
  FG_CHECK(v.shape() == ks, "attention: v must have k's shape " + shape_str(ks) + ", got " + shape_str(v.shape()));
  if (lengths)
    FG_CHECK(lengths->dtype() == DType::I32() && lengths->shape() == Shape{batch},
             "attention: the lengths must be i32 of shape " + shape_str(Shape{batch}) + ", got " + shape_str(lengths->shape()));
  FG_CHECK(std::isfinite(scale) && std::isfinite(static_cast<float>(scale)), "attention: scale must be finite");
  FG_CHECK(batch <= 0x7fffffffu && heads <= 0x7fffffffu, "attention: more than 2^31 - 1 sequences or heads");
  const size_t sq = qs[0] / batch, sk = ks[0] / batch;
  FG_CHECK(sq <= (1u << 28) && sk <= (1u << 28), "attention: sequences of more than 2^28 tokens");
  FG_CHECK(sq * (heads / kv_heads) <= (1u << 30), "attention: more than 2^30 queries of a sequence share a key head");
  need_hip(*this, "attention");
  const std::vector<int64_t> params = {static_cast<int64_t>(batch), static_cast<int64_t>(sq), static_cast<int64_t>(sk),
                                       static_cast<int64_t>(heads), static_cast<int64_t>(kv_heads),
                                       static_cast<int64_t>(dim), causal, lengths != nullptr, to_bits(scale)};
  std::vector<UOp> srcs = {source(uop()), source(k.uop()), source(v.uop())};
  if (lengths) srcs.push_back(source(lengths->uop()));
  srcs.push_back(output_storage(KernelId::Attention, 1, Shape{2, batch * heads * sq}, srcs, params));
  return from_uop(make_call(KernelId::Attention, qs, srcs, params), requires_grad() || k.requires_grad() || v.requires_grad());
}

Tensor Tensor::dropout(double p, uint64_t seed, uint64_t offset) const {
  FG_CHECK(dtype() == DType::F32(), "dropout: the input must be f32");
  FG_CHECK(p >= 0.0 && p < 1.0, "dropout: p must be in [0, 1), got " + std::to_string(p));
  FG_CHECK(numel() > 0, "dropout: the input is empty");
  need_hip(*this, "dropout");
  if (p == 0.0) return *this;
  const DeviceId d = device();
  return from_uop(make_call(KernelId::Dropout, shape(), {source(uop()), word(seed, d), word(seed >> 32, d), word(offset, d),
                                                         word(offset >> 32, d)},
                            {to_bits(p)}),
                  requires_grad());
}

Tensor Tensor::embedding(const Tensor& ids, double scale) const {
  FG_CHECK(dtype() == DType::F32(), "embedding: the weight must be f32");
  FG_CHECK(ndim() == 2, "embedding: the weight must be 2D (one row per id), got shape " + shape_str(shape()));
  FG_CHECK(numel() > 0, "embedding: the weight is empty");
  FG_CHECK(ids.dtype() == DType::I32() && ids.ndim() == 1,
           "embedding: the ids must be i32 of one dimension, got shape " + shape_str(ids.shape()));
  FG_CHECK(ids.numel() > 0, "embedding: the ids are empty");
  FG_CHECK(device() == ids.device(), "embedding: all tensors must be on the same device");
  FG_CHECK(std::isfinite(scale) && std::isfinite(static_cast<float>(scale)), "embedding: scale must be finite");
  const Shape s = shape();
  const size_t tokens = ids.numel();
  // Sizes that the kernels count in 32 bits, some workgroups' past the last.
  FG_CHECK(s[0] <= (1u << 30) && s[1] <= (1u << 30) && tokens <= (1u << 30), "embedding: more than 2^30 rows, columns or ids");
  need_hip(*this, "embedding");
  return from_uop(make_call(KernelId::Embedding, Shape{tokens, s[1]}, {source(uop()), source(ids.uop())},
                            {static_cast<int64_t>(tokens), static_cast<int64_t>(s[0]), static_cast<int64_t>(s[1]), to_bits(scale)}),
                  requires_grad());
}

Tensor Tensor::layer_norm(const Tensor& weight, const Tensor* bias, double eps) const {
  check_matrix(*this, "layer_norm: the input");
  FG_CHECK(device() == weight.device() && (!bias || device() == bias->device()), "layer_norm: all tensors must be on the same device");
  const Shape s = shape();
  for (const Tensor* t : {&weight, bias})
    if (t)
      FG_CHECK(t->dtype() == DType::F32() && t->shape() == Shape{s[1]},
               std::string("layer_norm: the ") + (t == bias ? "bias" : "weight") + " must be f32 of shape " +
                   shape_str(Shape{s[1]}) + ", got " + shape_str(t->shape()));
  // As float32, which the kernels add: infinity would give 0, and 0 NaN for a row of equal numbers.
  FG_CHECK(eps >= 0 && std::isfinite(static_cast<float>(eps)) && (eps == 0 || static_cast<float>(eps) > 0),
           "layer_norm: eps must be finite and not negative, and not 0 in float32 unless it is 0");
  FG_CHECK(s[0] <= (1u << 29) && s[1] <= (1u << 29), "layer_norm: more than 2^29 rows or columns");
  need_hip(*this, "layer_norm");
  std::vector<UOp> srcs = {source(uop()), source(weight.uop())};
  if (bias) srcs.push_back(source(bias->uop()));
  return from_uop(make_call(KernelId::LayerNorm, s, srcs,
                            {static_cast<int64_t>(s[0]), static_cast<int64_t>(s[1]), bias != nullptr, to_bits(eps)}),
                  requires_grad() || weight.requires_grad() || (bias && bias->requires_grad()));
}

Tensor Tensor::token_cross_entropy(const Tensor& labels) const {
  check_matrix(*this, "token_cross_entropy: the logits");
  const Shape s = shape();
  FG_CHECK(device() == labels.device(), "token_cross_entropy: all tensors must be on the same device");
  FG_CHECK(labels.dtype() == DType::I32() && labels.shape() == Shape{s[0]},
           "token_cross_entropy: the labels must be i32 of shape " + shape_str(Shape{s[0]}) + ", got " + shape_str(labels.shape()));
  FG_CHECK(s[0] <= (1u << 29) && s[1] <= (1u << 29), "token_cross_entropy: more than 2^29 rows or classes");
  need_hip(*this, "token_cross_entropy");
  return from_uop(make_call(KernelId::TokenLoss, Shape{1}, {source(uop()), source(labels.uop())},
                            {static_cast<int64_t>(s[0]), static_cast<int64_t>(s[1])}),
                  requires_grad());
}

Tensor Tensor::global_norm(const std::vector<Tensor>& tensors) {
  int64_t blocks = 0;
  const UOp sums = square_sums(clip_sources(tensors, "global_norm"), &blocks);
  return from_uop(make_call(KernelId::NormOfSums, Shape{1}, {sums}, {blocks}), false);
}

std::pair<Tensor, std::vector<Tensor>> Tensor::clip_norm(const std::vector<Tensor>& tensors, double max_norm) {
  FG_CHECK(max_norm > 0 && std::isfinite(max_norm), "clip_norm: max_norm must be finite and positive");
  const std::vector<UOp> all = clip_sources(tensors, "clip_norm");
  int64_t blocks = 0;
  const UOp sums = square_sums(all, &blocks);
  Tensor norm;
  std::vector<Tensor> out;
  for (size_t first = 0; first < all.size(); first += kClipTensors) {
    const size_t count = std::min(kClipTensors, all.size() - first);
    std::vector<UOp> srcs(all.begin() + static_cast<std::ptrdiff_t>(first), all.begin() + static_cast<std::ptrdiff_t>(first + count));
    std::vector<int64_t> params{to_bits(max_norm), blocks, first == 0};
    for (const UOp& u : srcs) params.push_back(static_cast<int64_t>(fg::numel(u.shape())));
    // A further output is told from other calls' by its tensor, the sums (of
    // all tensors) and its place.
    srcs.push_back(sums);
    std::vector<UOp> storage;
    for (size_t i = 1; i < count; i++)
      storage.push_back(output_storage(KernelId::Clip, static_cast<int64_t>(first + i), srcs[i].shape(), {srcs[i], sums}, {to_bits(max_norm)}));
    if (first == 0) storage.push_back(output_storage(KernelId::Clip, 0, Shape{1}, {sums}, {to_bits(max_norm)}));
    srcs.insert(srcs.end(), storage.begin(), storage.end());
    const UOp call = make_call(KernelId::Clip, srcs[0].shape(), srcs, params);
    out.push_back(from_uop(call, false));
    for (size_t i = 1; i < count; i++) out.push_back(from_uop(output_of(storage[i - 1], call), false));
    if (first == 0) norm = from_uop(output_of(storage.back(), call), false);
  }
  return {norm, out};
}

std::vector<UOp> kernel_gradient(const UOp& call, const UOp& grad) {
  switch (static_cast<KernelId>(call.arg().a)) {
    case KernelId::NormRotate: {
      std::vector<UOp> srcs = call.srcs();
      srcs.push_back(gradient_source(grad));
      UOp dw = output_storage(KernelId::NormRotateGrad, 1, call.src(1).shape(), srcs, params_of(call));
      srcs.push_back(dw);
      UOp dx = make_call(KernelId::NormRotateGrad, call.src(0).shape(), srcs, params_of(call));
      return {dx, output_of(dw, dx), UOp()};
    }
    case KernelId::Attention: {
      const std::vector<int64_t> params = params_of(call);
      std::vector<UOp> srcs = {call.src(0), call.src(1), call.src(2), call, gradient_source(grad)};
      srcs.push_back(output_of(call.srcs().back(), call));
      if (params[7]) srcs.push_back(call.src(3));
      UOp dk = output_storage(KernelId::AttentionGrad, 1, call.src(1).shape(), srcs, params);
      UOp dv = output_storage(KernelId::AttentionGrad, 2, call.src(2).shape(), srcs, params);
      srcs.push_back(dk);
      srcs.push_back(dv);
      UOp dq = make_call(KernelId::AttentionGrad, call.src(0).shape(), srcs, params);
      std::vector<UOp> grads = {dq, output_of(dk, dq), output_of(dv, dq)};
      grads.resize(call.srcs().size());
      return grads;
    }
    case KernelId::Embedding: {
      const Shape weight = call.src(0).shape();
      return {make_call(KernelId::EmbeddingGrad, weight, {call.src(1), gradient_source(grad)}, params_of(call)), UOp()};
    }
    case KernelId::LayerNorm: {
      const std::vector<int64_t> params = params_of(call);
      std::vector<UOp> srcs = {call.src(0), call.src(1), gradient_source(grad)}, storage;
      for (size_t i = 1; i < call.srcs().size(); i++)
        storage.push_back(output_storage(KernelId::LayerNormGrad, static_cast<int64_t>(i), call.src(1).shape(), srcs, params));
      srcs.insert(srcs.end(), storage.begin(), storage.end());
      UOp dx = make_call(KernelId::LayerNormGrad, call.src(0).shape(), srcs, params);
      std::vector<UOp> grads{dx};
      for (const UOp& u : storage) grads.push_back(output_of(u, dx));
      return grads;
    }
    case KernelId::TokenLoss: {
      std::vector<int64_t> params = params_of(call);
      // Of a gradient of 1, the seed of a backward pass, the call makes the loss too.
      const bool joint = is_ones(grad);
      params.push_back(joint);
      UOp last = joint ? output_storage(KernelId::TokenLossGrad, 1, call.shape(), {call}, params) : gradient_source(grad);
      return {make_call(KernelId::TokenLossGrad, call.src(0).shape(), {call.src(0), call.src(1), last}, params), UOp()};
    }
    case KernelId::NormRotateGrad:
    case KernelId::AttentionGrad:
    case KernelId::EmbeddingGrad:
    case KernelId::LayerNormGrad:
    case KernelId::TokenLossGrad: break;  // no second gradients
    case KernelId::SquareSums:
    case KernelId::NormOfSums:
    case KernelId::Clip: break;  // none through a norm
    case KernelId::Dropout: {
      // The same words again: the mask is never stored.
      std::vector<UOp> srcs = call.srcs();
      srcs[0] = gradient_source(grad);
      return {UOp::make_new(Op::Kernel, call.dtype(), srcs, call.arg())};
    }
  }
  fail("gradient not implemented for this kernel");
}

UOp kernel_also_made(const UOp& call) {
  if (call.op() != Op::Kernel || static_cast<KernelId>(call.arg().a) != KernelId::TokenLossGrad || !params_of(call)[2]) return UOp();
  return call.srcs().back().src(0);
}

RenderedKernel render_hip_call(const UOp& call) {
  RenderedKernel rk;
  switch (static_cast<KernelId>(call.arg().a)) {
    case KernelId::Dropout: rk = render_dropout(call); break;
    case KernelId::NormRotate: rk = render_norm_rotate(call, false); break;
    case KernelId::NormRotateGrad: rk = render_norm_rotate(call, true); break;
    case KernelId::Attention: rk = render_attention(call, false); break;
    case KernelId::AttentionGrad: rk = render_attention(call, true); break;
    case KernelId::Embedding: rk = render_embedding(call, false); break;
    case KernelId::EmbeddingGrad: rk = render_embedding(call, true); break;
    case KernelId::LayerNorm: rk = render_layer_norm(call, false); break;
    case KernelId::LayerNormGrad: rk = render_layer_norm(call, true); break;
    case KernelId::TokenLoss: rk = render_token_loss(call, false); break;
    case KernelId::TokenLossGrad: rk = render_token_loss(call, true); break;
    case KernelId::SquareSums: rk = render_square_sums(call); break;
    case KernelId::NormOfSums: rk = render_norm_of_sums(call); break;
    case KernelId::Clip: rk = render_clip(call); break;
  }
  rk.name = rk.launches.at(0).func;
  rk.out_slot = 0;
  rk.out_count = numel(shape_of(call));
  rk.params.emplace_back(0, call.dtype());
  for (size_t i = 0; i < call.srcs().size(); i++) rk.params.emplace_back(static_cast<int>(i) + 1, call.src(i).dtype());
  return rk;
}

}  // namespace fg
