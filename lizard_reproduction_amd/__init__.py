"""MI355X-native (gfx950) Lizard attention hot path.

``lizard_reproduction_amd.kernels`` is the drop-in for the reference's
``kernels`` package: ``gla`` (chunked gated linear attention) and ``swa``
(sliding-window softmax with sink logits), forward and backward in bf16, on
hand-written HIP kernels behind the C ABI of ``_lib/liblizard_hip.so``.  Beside
them: ``ssm`` (selective state space scan), ``short_conv`` and ``group_norm``.
"""
from . import kernels
from .kernels import gla, group_norm, short_conv, ssm, swa

__all__ = ["kernels", "gla", "swa", "ssm", "short_conv", "group_norm"]
