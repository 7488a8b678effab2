"""Core API (drop-in for the anchor part of ``scmiac.modeling.scmiac``) and the
device-side consumer of the anchor table (loaders, contrastive loss, dense layer,
distillation from a teacher's top logits)."""
from .scmiac import find_anchors
from .loss import NTXentLoss2
from .dense import LinearAct, linear_act
from .distill import NeighborDistillLoss, TopKDistillLoss, top_logits, topk_distill
from .dataset import DeviceAnchorLoader, DeviceMultiOmicLoader, anchor_frame, make_loaders

__all__ = ["find_anchors", "NTXentLoss2", "DeviceAnchorLoader", "DeviceMultiOmicLoader", "anchor_frame", "make_loaders",
           "linear_act", "LinearAct", "top_logits", "topk_distill", "TopKDistillLoss", "NeighborDistillLoss"]
