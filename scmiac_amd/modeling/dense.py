"""The dense layer of an encoder with its epilogue, forward and backward in HIP kernels.

``linear_act(x, weight, bias, residual, activation)`` is ``act(x @ weight.T + bias) + residual``: the
layers of the training loop's encoders (50 -> 128 -> 64 -> 30), and the scores of cells against a table
of reference cells -- with ``bias = -|r|^2 / 2`` the softmax over those scores is the soft
neighbourhood of the Euclidean distance.  float32, float16 and bfloat16; sums and the epilogue are
in float32 and rounded once.
"""
from __future__ import annotations

import torch.nn as nn

from .. import _hip


def linear_act(x, weight, bias=None, residual=None, activation="none"):
    """``act(x @ weight.T + bias) + residual`` on the GPU.

    ``x [..., k]``, ``weight [n, k]``, ``bias [n]``, ``residual [..., n]``: all float32, float16 or bfloat16 and on
    one device (``torch.autocast`` casts none of them); the result has their type.  ``activation``: ``"none"``, ``"relu"``,
    ``"gelu"`` (with the error function) or ``"silu"``.  ``x``, ``weight`` and ``residual`` may be strided; in float32 the product
    is as exact as float32 sums allow.  What an infinity or a NaN reaches is not finite; a large float32 layer makes NaN
    of an infinity where smaller ones may keep it.

    Gradients of all four, each the same number beside others and alone.  In the half types backward reads the
    pre-activation and the gradient of it rounded to the type, as a layer of separate operations does.  Refused with an error:
    second derivatives, forward-mode derivatives, tracing (``torch.jit.trace``, ``torch.export``; ``torch.compile`` runs it
    as it is between its graphs)."""
    _hip._cuda_device(x, "x")
    act = _hip.ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(_hip.ACTIVATIONS)}")
    return _hip.torch_ops().linear_act(x, weight, bias, residual, act)


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
