"""Linear block ``act(x W^T + b) + residual`` over channels-last rows, with its gradient.

The pointwise counterpart of ``ConvBlock`` (blocks.py): a 1 x 1 x 1 convolution over NDHWC voxels is a
matrix product of the voxels' rows with the weight, and bias, activation and the residual's addition ride
on its epilogue (``ops.linear``).  Under autograd the backward pass is the hand-written one
(``ops.linear_backward``): first order, all four gradients.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor, nn
from torch.autograd import forward_ad

from .. import _lib as L
from .. import ops


def _act_code(mod: nn.Module):
    if isinstance(mod, nn.ReLU):
        return L.ACT_RELU, 0.0
    if isinstance(mod, nn.LeakyReLU):
        return L.ACT_LRELU, float(mod.negative_slope)
    if isinstance(mod, nn.Tanh):
        return L.ACT_TANH, 0.0
    if isinstance(mod, nn.GELU) and mod.approximate == "none":
        return L.ACT_GELU, 0.0
    if isinstance(mod, nn.SiLU):
        return L.ACT_SILU, 0.0
    if isinstance(mod, nn.Identity):
        return L.ACT_NONE, 0.0
    raise NotImplementedError(f"activation {mod} has no HIP kernel")


def _rows(t: Tensor, cols: int) -> Tensor:
    """``t`` [..., cols] as a matrix with contiguous rows (a view wherever its strides allow one)."""
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), cols)
    elif t.is_contiguous():
        return t
    if not t.is_contiguous():
        s = t.stride()
        if (cols > 1 and s[1] != 1) or (t.shape[0] > 1 and s[0] < cols):
            t = t.contiguous()
    return t


_autocasts = torch.is_autocast_enabled


def _autocast(*tensors):
    """The operands in autocast's dtype (float64 ones are left as they are, as torch leaves them)."""
    dt = torch.get_autocast_dtype("cuda")
    return [t.to(dt) if t is not None and t.dtype in L.DTYPES else t for t in tensors]


def fused_linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, residual: Tensor | None = None,
                 act: int = L.ACT_NONE, slope: float = 0.0) -> Tensor:
    """``act(x weight^T + bias) + residual``: x [..., k], weight [n, k], bias [n], residual of the result's
    shape [..., n]; all of one dtype (float32, bfloat16 or float16).  ``act``: an activation code
    (``_lib.ACT_NONE``, ``ACT_RELU``, ``ACT_LRELU`` with ``slope``, ``ACT_TANH``, ``ACT_GELU``, ``ACT_SILU``).
    Under ``torch.autocast("cuda")`` all four are cast to its dtype first, as ``torch.nn.functional.linear``'s operands
    are (the residual too: bias, activation and sum stay in 32 bits, the result is rounded to that dtype once).
    Differentiable once, in reverse mode.  A HIP graph that captures the backward pass must be the only autograd graph alive
    on its leaves (torch's own rule: their gradient accumulators belong to the stream they were made on)."""
    if _autocasts("cuda"):
        x, weight, bias, residual = _autocast(x, weight, bias, residual)
    xs, ws = x.shape, weight.shape
    if len(ws) != 2 or not xs or xs[-1] != ws[1]:
        raise ValueError(f"fused_linear: x {tuple(xs)} does not multiply weight {tuple(ws)}")
    if residual is not None and (len(residual.shape) != len(xs) or residual.shape[-1] != ws[0]
                                 or residual.shape[:-1] != xs[:-1]):
        raise ValueError(f"fused_linear: residual {tuple(residual.shape)} is not of the result's shape "
                         f"{(*xs[:-1], ws[0])}")
    if forward_ad._current_level >= 0:
        ops._no_tangents("fused_linear", x, weight, bias, residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _LinearFn.apply(x, weight, bias, residual, act, slope)
    k = ws[1]
    return _forward(x, _rows(x, k), _rows(weight, k), bias, residual, act, slope, None)[0]


def _forward(x, x2, w2, bias, residual, act, slope, preact):
    n = w2.shape[0]
    if residual is not None and residual.is_contiguous() and residual.dtype is x.dtype:
        y = torch.empty_like(residual)  # the same shape, and cheaper to ask for
    else:
        y = x.new_empty((*x.shape[:-1], n))
    args = ops._linear_forward(x2, w2, y if y.dim() == 2 else y.view(x2.shape[0], n),
                               bias if bias is None or bias.is_contiguous() else bias.contiguous(),
                               residual if residual is None else _rows(residual, n), act, slope, preact)
    return y, args


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, slope):
        n, k = weight.shape
        x2, w2, preact = _rows(x, k), _rows(weight, k), None
        if act != L.ACT_NONE and True in ctx.needs_input_grad[:3]:
            preact = torch.empty((x2.shape[0], n), dtype=ops.linear_preact_dtype(x.dtype), device=x.device)
        y, ctx.args = _forward(x, x2, w2, bias, residual, act, slope, preact)
        ctx.shape, ctx.act, ctx.slope = x.shape, act, slope
        ctx.bias_shape = None if bias is None else bias.shape
        ctx.strides = x2.stride(), w2.stride()
        ctx.save_for_backward(x2, w2, preact)
        return y

    @staticmethod
    def backward(ctx, grad_out):
        if torch.is_grad_enabled():
            raise NotImplementedError("double backward through the HIP linear block is not implemented")
        if forward_ad._current_level >= 0:
            ops._no_tangents("fused_linear's backward pass", grad_out)
        x2, w2, preact = ctx.saved_tensors
        nx, nw, nb, nr = ctx.needs_input_grad[:4]
        dx = dw = None
        if nx:
            dx = torch.empty_like(x2) if x2.shape == ctx.shape and x2.is_contiguous() else x2.new_empty(ctx.shape)
        if nw:
            dw = torch.empty_like(w2) if w2.is_contiguous() else w2.new_empty(w2.shape)
        db = x2.new_empty(w2.shape[0]) if nb else None
        if nx or nw or nb:
            a, dy = ctx.args, _rows(grad_out, w2.shape[0])
            here = (x2.data_ptr() or None, w2.data_ptr() or None, None if preact is None else preact.data_ptr() or None)
            if (here == (a.x, a.w, a.preact) and (x2.stride(), w2.stride()) == ctx.strides
                    and (preact is None or preact.is_contiguous())):
                ops._linear_backward_of(a, dy, x2, dx, dw, db)
            else:  # hooks on saved tensors gave others back: elsewhere, or where the freed ones were with other strides
                ops.linear_backward(dy, _rows(x2, w2.shape[1]), _rows(w2, w2.shape[1]),
                                    dx if dx is None or dx.dim() == 2 else dx.view(x2.shape), dw, db, ctx.act, ctx.slope,
                                    preact if preact is None else preact.contiguous())
        if nb and db.shape != ctx.bias_shape:  # n values in any shape
            db = db.view(ctx.bias_shape)
        return dx, dw, db, grad_out if nr else None, None, None


class LinearBlock(nn.Module):
    """``activation_fn(linear(x)) + residual`` on channels-last tensors [..., channels_in]: parameters in
    ``nn.Linear``'s layout under ``linear``."""

    def __init__(self, channels_in: int, channels_out: int, activation_fn: type = nn.ReLU, bias: bool = True, **kwargs):
        super().__init__()
        self.linear = nn.Linear(channels_in, channels_out, bias=bias)
        self.activation_fn = activation_fn(**kwargs)
        _act_code(self.activation_fn)  # refuse what has no kernel where the block is built

    def forward(self, x: Tensor, residual: Tensor | None = None) -> Tensor:
        act, slope = _act_code(self.activation_fn)
        return fused_linear(x, self.linear.weight, self.linear.bias, residual, act, slope)
