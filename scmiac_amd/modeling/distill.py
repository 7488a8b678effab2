"""Learning from a teacher's top logits: the teacher's table and the loss, in HIP kernels.

``top_logits`` cuts a teacher's scores down to the k best classes of each row and their normaliser;
``topk_distill`` is the loss (and gradient) of a student's logits against such a table.  A k-NN
table is one, too: ``idx`` and ``-dist2`` of :func:`scmiac_amd._hip.knn_search`, padding included.
``NeighborDistillLoss`` puts the two together for embeddings, next to ``NTXentLoss2``: the soft
neighbours a teacher's table lists instead of one positive per row.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .. import _hip
from .dense import linear_act


def top_logits(logits, k, temperature=1.0):
    """The ``k`` (at most 64) largest logits of each row, by value and, where equal, by index.

    Returns ``(values [..., k], idx [..., k] int32, lse [...] float32)``; ``values`` has the logits' type,
    ``lse`` is ``log sum exp(logits / temperature)`` over the whole row.  Rows of fewer than ``k`` classes are padded
    with ``-inf`` and -1; of a row with a NaN ``lse`` is NaN and the entries are unspecified.  No derivative flows: a teacher is a
    constant.  Cannot be traced."""
    _hip._cuda_device(logits, "logits")
    return _hip.torch_ops().top_logits(logits, int(k), temperature)


def topk_distill(logits, teacher_idx, teacher_logits, temperature=1.0, teacher_lse=None, teacher_temperature=None,
                 reduction="mean"):
    """Distillation from a teacher's top logits:
    ``sum_i t_i (log t_i - log_softmax(logits / temperature)[idx_i])`` per row, with
    ``t = softmax(teacher_logits / teacher_temperature)`` over the listed classes or, given ``teacher_lse`` (the
    teacher's log-sum-exp at that temperature over all its classes), ``exp(teacher_logits / teacher_temperature -
    teacher_lse)``.  No factor ``temperature ** 2``.

    ``logits [..., v]`` float32, float16 or bfloat16, rows may be strided; ``teacher_idx [..., k]`` (k at most 1024)
    whole numbers, -1 for padding, a class may be listed twice; ``teacher_logits [..., k]``; ``teacher_temperature``
    defaults to ``temperature``.  ``reduction``: ``"none"``, ``"sum"`` or ``"mean"`` over the rows that have a teacher: rows
    of padding only or of teacher logits that are all ``-inf``, whatever the student's logits hold, and rows of student
    logits that are all ``-inf`` have loss and gradient 0 and are left out.  An index that is no class makes its row's loss
    and gradient NaN (nothing waits for the GPU to raise).  Gradients for ``logits`` alone: the teacher has to be detached.
    Second derivatives, forward-mode derivatives and tracing are refused."""
    _hip._cuda_device(logits, "logits")
    number = _hip.REDUCTIONS.get(reduction)
    if number is None:
        raise ValueError(f"reduction must be one of {sorted(_hip.REDUCTIONS)}")
    if teacher_temperature is None:
        teacher_temperature = temperature
    return _hip.torch_ops().topk_distill(logits, teacher_idx, teacher_logits, teacher_lse, temperature, teacher_temperature,
                                         number)


class TopKDistillLoss(nn.Module):
    """:func:`topk_distill` as a module: ``loss(logits, teacher_idx, teacher_logits, teacher_lse=None)``."""

    def __init__(self, temperature=1.0, teacher_temperature=None, reduction="mean"):
        super().__init__()
        self.temperature, self.teacher_temperature, self.reduction = temperature, teacher_temperature, reduction

    def forward(self, logits, teacher_idx, teacher_logits, teacher_lse=None):
        return topk_distill(logits, teacher_idx, teacher_logits, self.temperature, teacher_lse, self.teacher_temperature,
                            self.reduction)


def _unit(z):
    """Rows of length 1, worked out in float32.  Rows of zeros stay zeros: in float16 1e-12, what they are divided by
    in float32, would be 0, and their gradients too large; it is the smallest normal number there."""
    eps = max(1e-12, torch.finfo(z.dtype).smallest_normal)
    return nn.functional.normalize(z.float(), dim=-1, eps=eps).to(z.dtype)


class NeighborDistillLoss(nn.Module):
    """Soft-neighbour loss of embeddings: ``loss(z, z_ref, teacher_idx, teacher_logits)`` compares the softmax of the
    similarities of ``z [n, d]`` to all of ``z_ref [m, d]`` with the neighbours the table ``teacher_idx [n, k]`` lists
    (rows of ``z_ref``, -1 for padding) at weights ``softmax(teacher_logits / teacher_temperature)``, for instance
    ``idx`` and ``-dist2`` of a k-NN search.

    ``metric="cosine"`` (as ``NTXentLoss2``): ``z . z_ref / temperature`` of rows normalised to length 1;
    ``"euclidean"``: ``-|z - z_ref|^2 / (2 temperature)``.  Gradients for ``z`` and ``z_ref``.  The scores are stored
    (n x m, in the embeddings' type): made for batches of cells against a reference set."""

    def __init__(self, temperature=0.5, teacher_temperature=1.0, metric="cosine", reduction="mean"):
        super().__init__()
        if metric not in ("cosine", "euclidean"):
            raise ValueError("metric must be 'cosine' or 'euclidean'")
        self.temperature, self.teacher_temperature = temperature, teacher_temperature
        self.metric, self.reduction = metric, reduction

    def forward(self, z, z_ref, teacher_idx, teacher_logits, teacher_lse=None):
        bias = None
        if self.metric == "cosine":
            z, z_ref = _unit(z), _unit(z_ref)
        else:  # the softmax over the references does not see |z|^2 (float16 has no squares from 256 on: their sum is float32)
            bias = (-0.5 * z_ref.float().square().sum(-1)).to(z_ref.dtype)
        return topk_distill(linear_act(z, z_ref, bias), teacher_idx, teacher_logits, self.temperature, teacher_lse,
                            self.teacher_temperature, self.reduction)
