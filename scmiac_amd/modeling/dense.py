"""The dense layer of an encoder with its epilogue, forward and backward in HIP kernels.

``linear_act(x, weight, bias, residual, activation)`` is ``act(x @ weight.T + bias) + residual``: the
layers of the training loop's encoders (50 -> 128 -> 64 -> 30), and the scores of cells against a table
of reference cells -- with ``bias = -|r|^2 / 2`` the softmax over those scores is the soft
neighbourhood of the Euclidean distance.  float32, float16 and bfloat16; sums and the epilogue are
in float32 and rounded once.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import _hip


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        need = ctx.needs_input_grad
        keep = need[0] or need[1] or need[2]
        y, z = _hip.linear_forward(x, weight, bias, residual, activation, keep_z=keep)
        ctx.activation = activation
        ctx.k = x.shape[1]
        if keep:
            ctx.save_for_backward(x if need[1] else None, weight if need[0] else None, z)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0] or need[1] or need[2]:
            x, weight, z = ctx.saved_tensors
            dx, dw, db = _hip.linear_backward(x, weight, z, dy, ctx.k, ctx.activation, need[:3])
        return dx, dw, db, dy if need[3] else None, None


def linear_act(x, weight, bias=None, residual=None, activation="none"):
    """``act(x @ weight.T + bias) + residual`` on the GPU.

    ``x [..., k]``, ``weight [n, k]``, ``bias [n]``, ``residual [..., n]``: all float32, float16 or bfloat16 and on
    one device; the result has their type.  ``activation``: ``"none"``, ``"relu"``, ``"gelu"`` (with the error
    function) or ``"silu"``.  Gradients of all four; not differentiable twice.  ``x``, ``weight`` and ``residual``
    may be strided; in float32 the product is as exact as float32 sums allow."""
    device = _hip._cuda_device(x, "x")
    _hip.load_library()
    if x.dtype not in _hip.DTYPES:
        raise TypeError(f"linear_act expects float32, float16 or bfloat16, not {x.dtype}")
    if activation not in _hip.ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_hip.ACTIVATIONS)}")
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is None and name != "weight":
            continue
        if _hip._cuda_device(t, name) != device:
            raise ValueError(f"{name} is on {t.device}, x on {device}")
        if t.dtype != x.dtype:
            raise TypeError(f"{name} is {t.dtype}, x is {x.dtype}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"x [..., k] and weight [n, k] do not match: {tuple(x.shape)}, {tuple(weight.shape)}")
    shape = x.shape[:-1] + weight.shape[:1]
    if bias is not None and bias.shape != shape[-1:]:
        raise ValueError(f"bias needs shape {tuple(shape[-1:])}, not {tuple(bias.shape)}")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"residual needs shape {tuple(shape)}, not {tuple(residual.shape)}")
    flat = x.dim() == 2
    x2 = x if flat else x.reshape(-1, x.shape[-1])
    r2 = residual if flat or residual is None else residual.reshape(-1, shape[-1])
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        y = _LinearAct.apply(x2, weight, bias, r2, activation)
    else:
        y = _hip.linear_forward(x2, weight, bias, r2, activation)[0]
    return y if flat else y.view(shape)


class LinearAct(nn.Linear):
    """``torch.nn.Linear`` (same parameters and initialisation) with the activation and an optional
    residual in the product's epilogue: ``layer(x, residual=None)``."""

    def __init__(self, in_features, out_features, bias=True, activation="none", device=None, dtype=None):
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        if activation not in _hip.ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(_hip.ACTIVATIONS)}")
        self.activation = activation

    def forward(self, x, residual=None):
        return linear_act(x, self.weight, self.bias, residual, self.activation)

    def extra_repr(self):
        return f"{super().extra_repr()}, activation={self.activation!r}"
