// Hand-written kernels behind Tensor methods: attention, per-head norms with
// the position rotation, dropout; embedding, layer norm, the loss of token
// labels, and clipping to a global norm. No reference counterpart: the
// reference composes every op out of its IR, which has no random numbers, no
// sine, no indexing by data and only two-dimensional products.
//
// A call is one Op::Kernel node whose sources are its arguments: matrices read
// as whole buffers (the scheduler gives what computes them a kernel of its
// own), integers that change from call to call as I32 constants (left out of
// the realisation plan's key, like Shrink starts), and an Op::KernelBuf for
// every output after the first. Its Arg holds the KernelId, the first output's
// shape and the parameters that pick variants and geometry.
#pragma once

#include "device.hpp"
#include "ir.hpp"

namespace fg {

enum class KernelId : int64_t {
  Dropout = 0, NormRotate, NormRotateGrad, Attention, AttentionGrad, Embedding, EmbeddingGrad, LayerNorm, LayerNormGrad,
  TokenLoss, TokenLossGrad, SquareSums, NormOfSums, Clip
};

// The gradients of a call's sources (null where there is none), for
// gradient_for_op.
std::vector<UOp> kernel_gradient(const UOp& call, const UOp& grad);

// The other call whose result `call` makes as well, in the storage that is its
// last source (of the loss of token labels, its gradient does), or null. That
// storage has the other call as its source, so a graph that has `call` has both.
UOp kernel_also_made(const UOp& call);

// The launches of a call on the MI355X (Device::render_call): functions of the
// library's code object, their geometry and arguments.
RenderedKernel render_hip_call(const UOp& call);

}  // namespace fg
