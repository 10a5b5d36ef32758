"""DPGroupNorm: group norm with per-sample-clipped, noised dgamma / dbeta, and the activation and dropout behind it.

No counterpart in the reference, whose layers are Linear, Conv1D and LayerNorm.  Group norm is what networks over images and
patches use under DP-SGD in the place of batch norm, whose statistics mix the samples of a batch.
"""
import torch
import torch.nn as nn
from torch.autograd.function import Function, once_differentiable

from ..core import ops
from .utils import DPParameter as Parameter
from ._common import DPLayerMixin, dp_scalars, dropout_spec, leaves_a_graph


def _channels_first(t):
    """(B, *, C) as a contiguous (B, C, *) of its own"""
    t = t.movedim(-1, 1)
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


class _DPGroupNormFunc(Function):
    @staticmethod
    def forward(ctx, input, weight, bias, layer, spec, channels_first):
        """`channels_first`: input, output and the input's gradient are contiguous (B, C, *)."""
        x = input.movedim(1, -1) if channels_first else input
        x = x.contiguous()                    # (so that the backward does not copy it once more)
        y, stats = ops.group_norm_forward(x, weight, bias, layer.num_groups, layer.eps, activation=layer.activation, dropout=spec)
        ctx.save_for_backward(x, weight, bias, stats["mean"], stats["rstd"])
        ctx.layer, ctx.spec, ctx.activation, ctx.channels_first = layer, spec, layer.activation, channels_first
        return _channels_first(y) if channels_first else y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        input, weight, bias, mean, rstd = ctx.saved_tensors
        layer = ctx.layer
        B = input.shape[0]
        div, noise = dp_scalars(B, layer.noise_multiplier, layer._dp_param_ids[0], layer._next_step(),
                                param_id2=layer._dp_param_ids[1])
        need_dw = weight is not None and (ctx.needs_input_grad[1] or ctx.needs_input_grad[2])
        if ctx.channels_first:
            grad_output = grad_output.movedim(1, -1)
        dx, dw, db = ops.dp_group_norm_backward(
            grad_output, input, weight, bias, mean, rstd, layer.num_groups, layer.C, layer.clamp_value,
            activation=ctx.activation, dropout=ctx.spec, batch_divisor=div, noise=noise, need_dx=ctx.needs_input_grad[0],
            need_dw=need_dw)
        if ctx.channels_first and dx is not None:
            dx = _channels_first(dx)
        return dx, dw if ctx.needs_input_grad[1] else None, db if ctx.needs_input_grad[2] else None, None, None, None


class DPGroupNorm(nn.GroupNorm, DPLayerMixin):
    """nn.GroupNorm over (B, C, *), with `activation` (None, "relu", "silu", "gelu" or "gelu_tanh") and `dropout` (the
    probability; in training only) behind it in the same kernels.  They work on channels-last storage: an input in
    torch.channels_last (or channels_last_3d) is taken as it lies, and output and input gradient have that format too.  For any
    other they are contiguous, as nn.GroupNorm's, at the price of a copy of each of the input, the output and their gradients.
    `channels_last=True`: input and output are (B, *, C), as those of the Linear layers, and nothing is copied.  (16 x 320 x 64 x 64 bf16 with silu, forward and backward: 106 us in channels_last, 434 contiguous; 8 x 256 x 128 x 128 fp32 190
    and 760.)  The output has the input's type, under autocast too."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True, device=None, dtype=None,
                 activation=None, dropout: float = 0.0, channels_last: bool = False, C: float = 1.0, clamp_value: float = 1.0,
                 noise_multiplier: float = 1.0):
        super().__init__(num_groups, num_channels, eps, affine, device=device, dtype=dtype)
        ops._activation(activation)
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"dropout probability has to be between 0 and 1, but got {dropout}")
        self.activation, self.dropout, self.channels_last = activation, float(dropout), bool(channels_last)
        self._init_dp(C, clamp_value, noise_multiplier, n_tensors=3)      # gamma, beta, the dropout's stream
        if affine:
            self.weight = Parameter(self.weight.data)
            self.bias = Parameter(self.bias.data)

    def forward(self, input):
        if input.dim() < 2 or input.shape[-1 if self.channels_last else 1] != self.num_channels:
            raise RuntimeError(f"expected {'(B, *, C)' if self.channels_last else '(B, C, *)'} with C = {self.num_channels}, "
                               f"got {tuple(input.shape)}")
        x = input if self.channels_last else input.movedim(1, -1)
        spec = None
        if self.training and self.dropout > 0.0:
            spec = dropout_spec(self.dropout, self._dp_param_ids[2], x, leaves_a_graph(x, self.weight, self.bias))
        if self.channels_last:
            return _DPGroupNormFunc.apply(x, self.weight, self.bias, self, spec, False)
        if x.is_contiguous() and (input.dim() in (4, 5) or input.is_contiguous()):      # (of three axes there is no such format)
            return _DPGroupNormFunc.apply(x, self.weight, self.bias, self, spec, False).movedim(-1, 1)
        return _DPGroupNormFunc.apply(input, self.weight, self.bias, self, spec, True)

    def extra_repr(self):
        return f"{super().extra_repr()}, activation={self.activation}, dropout={self.dropout}"
