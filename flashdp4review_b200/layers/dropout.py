"""DPDropout: nn.Dropout whose mask is drawn from a counter-based generator in the kernels, forward and backward, and never
stored; the residual sum behind it is part of the call.  No counterpart in the reference, whose models use nn.Dropout.
"""
import torch
import torch.nn as nn
from torch.autograd.function import Function, once_differentiable

from .. import runtime
from ..core import ops
from ._common import dropout_spec, leaves_a_graph


def _storage_order(x):
    """The axes of a dense tensor from the slowest to the fastest, so that channels-last storage is walked as it lies."""
    order = sorted(range(x.dim()), key=lambda d: (-x.stride(d), d))
    return order if x.permute(order).is_contiguous() else list(range(x.dim()))


class _InPlace(Function):
    """Autograd's own check that `input` may be modified, which it makes behind a Function's forward: here before anything is."""
    @staticmethod
    def forward(ctx, input):
        ctx.mark_dirty(input)
        return input

    @staticmethod
    def backward(ctx, grad_output):
        return grad_output


class _DropoutFunc(Function):
    @staticmethod
    def forward(ctx, input, residual, spec, inplace):
        # elements are numbered in the order of the input's storage; the gradient is brought into the same one
        ctx.order, ctx.spec = _storage_order(input), spec
        x = input.permute(ctx.order)
        if inplace:
            if x.is_contiguous():
                ops.dropout(x, spec, out=x)
            else:
                input.copy_(ops.dropout(x, spec))           # (its axes are in order)
            ctx.mark_dirty(input)
            return input
        if ctx.order == sorted(ctx.order):
            return ops.dropout(x, spec, residual=residual)
        # a tensor of the input's strides, written through a permuted view: a view that the Function returned could not be modified in place
        y = torch.empty_strided(input.shape, input.stride(), dtype=input.dtype, device=input.device)
        ops.dropout(x, spec, residual=None if residual is None else residual.permute(ctx.order), out=y.permute(ctx.order))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        dx = None
        if ctx.needs_input_grad[0]:
            dx = ops.dropout_backward(grad_output.permute(ctx.order), ctx.spec).permute(_inverse(ctx.order))
        return dx, grad_output if ctx.needs_input_grad[1] else None, None, None


def _inverse(order):
    inverse = [0] * len(order)
    for i, d in enumerate(order):
        inverse[d] = i
    return inverse


class DPDropout(nn.Dropout):
    """`forward(input)` drops as nn.Dropout does; `forward(input, residual)` adds `residual`, in the same kernel where it has the
    input's type and shape and with an ordinary sum where not (a 16-bit branch onto an fp32 residual under autocast).  In
    evaluation mode, and for p = 0, the input (or the sum) comes back.  The mask's seed is drawn from torch's CPU generator:
    torch.manual_seed repeats a run, and torch.utils.checkpoint, which restores that generator, draws a recomputed pass's
    mask again.  With use_device_noise_step() on, such a pass is known by its seed: two graphs that drew from one seed at
    different steps cannot be told apart, and running one of them again is refused.  Data-parallel ranks draw for their own
    shards, whatever their sizes.  In a captured step use_device_noise_step() has to be on (every replay then draws anew), else
    the call is refused."""

    def __init__(self, p: float = 0.5, inplace: bool = False):
        super().__init__(p, inplace)
        self._stream_id = runtime.next_dropout_id()

    def forward(self, input, residual=None):
        if not self.training or self.p == 0.0:
            return input if residual is None else input + residual
        if self.inplace and residual is not None:
            raise RuntimeError("dropout in place takes no residual")
        if residual is not None and not (torch.is_tensor(residual) and residual.shape == input.shape and residual.dtype == input.dtype
                                         and residual.device == input.device):
            return self.forward(input) + residual
        graph = leaves_a_graph(input, residual)
        if self.inplace and graph:
            input = _InPlace.apply(input)
        y = _DropoutFunc.apply(input, residual, dropout_spec(self.p, self._stream_id, input, graph), self.inplace)
        return input if self.inplace and not graph else y         # (a leaf without a graph comes back as itself)
