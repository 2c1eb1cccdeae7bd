// Hand-written kernels behind Tensor methods: attention, per-head norms with
// the position rotation, dropout. No reference counterpart: the reference
// composes every op out of its IR, which has no random numbers, no sine and
// only two-dimensional products.
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

enum class KernelId : int64_t { Dropout = 0, NormRotate, NormRotateGrad, Attention, AttentionGrad };

// The gradients of a call's sources (null where there is none), for
// gradient_for_op.
std::vector<UOp> kernel_gradient(const UOp& call, const UOp& grad);

// The launches of a call on the MI355X (Device::render_call): functions of the
// library's code object, their geometry and arguments.
RenderedKernel render_hip_call(const UOp& call);

}  // namespace fg
