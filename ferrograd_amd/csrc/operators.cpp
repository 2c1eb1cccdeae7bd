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
    case KernelId::NormRotateGrad:
    case KernelId::AttentionGrad: break;  // no second gradients
    case KernelId::Dropout: {
      // The same words again: the mask is never stored.
      std::vector<UOp> srcs = call.srcs();
      srcs[0] = gradient_source(grad);
      return {UOp::make_new(Op::Kernel, call.dtype(), srcs, call.arg())};
    }
  }
  fail("gradient not implemented for this kernel");
}

RenderedKernel render_hip_call(const UOp& call) {
  RenderedKernel rk;
  switch (static_cast<KernelId>(call.arg().a)) {
    case KernelId::Dropout: rk = render_dropout(call); break;
    case KernelId::NormRotate: rk = render_norm_rotate(call, false); break;
    case KernelId::NormRotateGrad: rk = render_norm_rotate(call, true); break;
    case KernelId::Attention: rk = render_attention(call, false); break;
    case KernelId::AttentionGrad: rk = render_attention(call, true); break;
  }
  rk.name = rk.launches.at(0).func;
  rk.out_slot = 0;
  rk.out_count = numel(shape_of(call));
  rk.params.emplace_back(0, call.dtype());
  for (size_t i = 0; i < call.srcs().size(); i++) rk.params.emplace_back(static_cast<int>(i) + 1, call.src(i).dtype());
  return rk;
}

}  // namespace fg
