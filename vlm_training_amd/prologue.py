"""The element-wise work either side of the attention operator, fused into single passes over HBM.

``qk_norm_rope``  replaces, in the reference's attention layers, ``q_norm(q)``/``k_norm(k)`` (F.rms_norm per
head), the transpose to (B, H, S, D), ``apply_rope``, the transpose back and the ``.contiguous()`` copies
(models/qwen3_vl/model.py:256-269; models/qwen3_5/model.py:110-129 with OffsetRMSNorm and a partial
rotary width): the projections' outputs go in as (T, H, D) *views* (any token / head stride, so the q
half of Qwen3.5's interleaved ``[q | gate]`` projection is read in place), the packed (T, H, D) tensors
the attention operator wants come out.  ``sigmoid_gate`` is ``out * torch.sigmoid(gate)``
(models/qwen3_5/model.py:135).  ``gated_rms_norm`` is the norm behind a block with its SiLU gate (models/qwen3_5/model.py:38-44),
``residual_rms_norm`` the residual addition between two blocks with the next one's norm.  All are autograd nodes in csrc/dsa_host.cpp and
csrc/dsa_host_layer.cpp over the C ABI; there is no fallback path.
"""
from __future__ import annotations

import torch

from . import _lib


@torch.compiler.disable
def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, eps: float = 1e-6, offset: bool = False):
    """q (T, Hq, D), k (T, Hkv, D) bf16 views -> rope(rms_norm(q)), rope(rms_norm(k)) as contiguous (T, H, D).

    ``offset=True`` scales by ``1 + weight`` (OffsetRMSNorm).  cos, sin: (T, R) or (1, T, R), R <= D a
    multiple of 16 (elements past R pass through unrotated)."""
    return tuple(_lib.host().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, float(eps), bool(offset)))


@torch.compiler.disable
def sigmoid_gate(x, gate):
    """``x * torch.sigmoid(gate)`` for x (T, H, D) contiguous and gate a (T, H, D) view (strided allowed)."""
    return _lib.host().sigmoid_gate(x, gate)


@torch.compiler.disable
def gated_rms_norm(x, gate, weight, eps: float = 1e-6, offset: bool = False):
    """``rms_norm(x) * weight * silu(gate)`` per row of D for x, gate (T, H, D) bf16 views, D a multiple of 8 up to 512; ``offset=True`` scales by
    ``1 + weight``.  Second derivatives raise."""
    return _lib.host().gated_rms_norm(x, gate, weight, float(eps), bool(offset))


@torch.compiler.disable
def residual_rms_norm(x, y, weight, *, post_weight=None, gate=None, scale=None, eps: float = 1e-6, offset: bool = False):
    """The residual stream ``x`` and a block's output ``y`` (..., C) -> (the stream behind the block, the next block's input):

    ``x' = x + scale * sigmoid(gate) * [rms_norm(y) * post_weight]``, ``h = rms_norm(x') * weight``.  ``post_weight`` (C,) norms the block's output before it
    is added, ``gate`` (..., C) and ``scale`` (a number, or (C,)) weigh it; each may be left out.  x is bf16 or fp32 and so is x'; y, gate
    and h are bf16; C is a multiple of 8 up to 8192; ``offset=True`` scales by ``1 + weight`` in both norms.  The norm reads x' before it is rounded, and its
    gradients are taken there: for them a bf16 stream's x and y are kept, of an fp32 stream x' (and y where one of the three is given).  Second
    derivatives raise."""
    if isinstance(scale, (int, float)):
        scale = torch.full(x.shape[-1:], float(scale), dtype=torch.float32, device=x.device)
    return tuple(_lib.host().residual_rms_norm(x, y, weight, post_weight, gate, scale, float(eps), bool(offset)))
