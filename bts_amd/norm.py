"""Layer normalisation with autograd on the HIP kernels `bts_layernorm_fwd` / `bts_layernorm_bwd`.

The decoder normalises with BatchNorm (bts.py:155-172), whose statistics are taken over the images of ONE rank; layer normalisation does
not depend on the batch.  ``LayerNorm`` takes the place of ``torch.nn.LayerNorm`` (same arguments, parameters and state-dict keys),
``LayerNorm2d`` normalises the channels at every pixel of an NCHW map, where ``nn.BatchNorm2d`` would normalise the batch.

Inputs are f32 or bf16, parameters and their gradients f32, statistics f32; the result has the input's type, also under autocast (where
``torch.nn.LayerNorm`` gives f32 for a bf16 input), and ``module.bfloat16()`` makes parameters that are refused.  No second and no
forward-mode derivatives, no torch.jit.trace (all refused), no CPU path.
"""
import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import ops
from ._lib import BtsAmdError

_is_tracing = torch._C._is_tracing

__all__ = ["layer_norm", "LayerNorm", "LayerNorm2d"]


def _rows(t):
    """t itself where the kernels can walk it (contiguous, evenly strided rows), else a dense copy; and what row_stride says of it."""
    rows = ops.row_stride(t)
    if rows is None:
        t = t.contiguous()
        rows = ops.row_stride(t)
    return t, rows


def _backward(ctx, dy):
    x, weight = ctx.saved_tensors
    need = ctx.needs_input_grad
    dy, (_, dys) = _rows(dy)
    dev = dy.get_device()
    if x.stride() == ctx.strides and x.shape == dy.shape and x.dtype == dy.dtype and x.get_device() == dev and (
            weight is None or weight.dtype == torch.float32 and weight.is_contiguous() and weight.numel() == x.shape[-1] and weight.get_device() == dev):
        return (*ops.layer_norm_bwd_unchecked(dy, dys, x, ctx.rows, ctx.stats, weight, need[0], need[1], need[2]), None)
    # Saved-tensor hooks gave back other tensors than were saved (save_on_cpu: a slice of a wider buffer comes back dense): their own
    # layout counts, and what is not the saved values' shape, type and device is refused.
    weight = weight if weight is None else weight.contiguous()
    return (*ops.layer_norm_bwd(dy, _rows(x)[0], ctx.stats, weight, need[0], need[1], need[2]), None)


_backward_once = once_differentiable(_backward)


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x, rows = _rows(x)
        y, stats = ops.layer_norm_fwd_rows(x, rows, weight, bias, eps, True)
        ctx.save_for_backward(x, weight)
        ctx.rows, ctx.strides, ctx.stats = rows, x.stride(), stats           # (nobody else has the statistics: not for hooks to change)
        return y

    @staticmethod
    def backward(ctx, dy):
        # the engine hands over a gradient of y's shape, type and device, on y's device; a graph of this pass is only asked for with
        # create_graph, and refused where it would be differentiated
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x [..., C], 1 <= C <= 16384; weight and bias f32 [C] or None."""
    if x.dim() == 0:
        raise BtsAmdError("layer_norm: x must have at least one axis")
    if _is_tracing():
        raise BtsAmdError("layer_norm cannot be traced: torch.jit.trace would record the allocation of its result and no launch")
    # forward-mode differentiation sees the call only through the Function, which refuses a tangent (a dual tensor does not require gradients)
    if (torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad))
            or forward_ad._current_level >= 0):
        return _LayerNormFn.apply(x, weight, bias, float(eps))
    return ops.layer_norm_fwd_rows(*_rows(x), weight, bias, float(eps), False)


class LayerNorm(nn.LayerNorm):
    """``torch.nn.LayerNorm`` on the HIP kernels: normalises over the trailing axes `normalized_shape`.  The result has x's type; the
    parameters stay f32."""

    def forward(self, x):
        shape = tuple(self.normalized_shape)
        if tuple(x.shape[x.dim() - len(shape):]) != shape or x.dim() < len(shape):
            raise BtsAmdError("LayerNorm over %s got an input of shape %s" % (shape, tuple(x.shape)))
        if len(shape) == 1:
            return layer_norm(x, self.weight, self.bias, self.eps)
        flat = (t if t is None else t.reshape(-1) for t in (self.weight, self.bias))
        return layer_norm(x.flatten(x.dim() - len(shape)), *flat, self.eps).view(x.shape)


class LayerNorm2d(nn.LayerNorm):
    """Normalises the C channels at every pixel of x [N, C, H, W].  A channels-last map is read and written in place of its layout; a
    contiguous NCHW map costs a copy, and the result is channels-last either way."""

    def __init__(self, num_channels, eps=1e-5, elementwise_affine=True, **kw):
        super().__init__(num_channels, eps=eps, elementwise_affine=elementwise_affine, **kw)

    def forward(self, x):
        if x.dim() != 4 or x.shape[1] != self.normalized_shape[0]:
            raise BtsAmdError("LayerNorm2d over %d channels got an input of shape %s" % (self.normalized_shape[0], tuple(x.shape)))
        return layer_norm(x.permute(0, 2, 3, 1), self.weight, self.bias, self.eps).permute(0, 3, 1, 2)
