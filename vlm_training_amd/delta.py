"""The token mixer of the linear-attention layers in the reference's hybrid stack: a short convolution and the gated delta rule.

``short_conv``        depthwise causal convolution with SiLU over packed sequences (models/qwen3_5/model.py:173-176), ``short_conv_step`` for one
                      token of each request.
``gated_delta_rule``  runs packed sequences in chunks (models/qwen3_5/model.py:178-186: ``q``, ``k`` normalised inside, decay and write strength
                      from the projections ``a``, ``b`` and the parameters ``a_log``, ``dt_bias``), with gradients for every input, from and to states.
``gated_delta_step``  one token for each of a batch of requests, the states updated in place (decoding).

Per value head a state ``S`` (Dk, Dv) in fp32, with ``g = -exp(a_log) * softplus(a + dt_bias)`` and ``beta = sigmoid(b)``:
``S = exp(g) * S + beta * k (v - exp(g) * S^T k)^T``, ``o = scale * S^T q``.  Value head ``h`` reads key head ``h // (Hv // Hk)``.
Autograd nodes in csrc/dsa_host_layer.cpp over the C ABI; there is no fallback path.
"""
from __future__ import annotations

import torch

from . import _lib


@torch.compiler.disable
def gated_delta_rule(q, k, v, a, b, a_log, dt_bias, cu_seqlens, *, scale=None, l2_norm: bool = True, initial_state=None,
                     return_final_state: bool = False):
    """q, k (T, Hk, Dk), v (T, Hv, Dv) bf16 views, a, b (T, Hv), a_log, dt_bias (Hv,) bf16 or fp32 -> (T, Hv, Dv) bf16.

    Head dims are multiples of 8 up to 128.  ``scale`` defaults to ``Dk ** -0.5``; ``l2_norm=False`` takes q and k as they are.
    ``cu_seqlens`` (N+1,) are the packed sequences' offsets (empty ones allowed); rows behind the last sequence give zeros.  ``initial_state`` (N, Hv, Dk, Dv)
    fp32 is where the sequences start (zeros without one); with ``return_final_state`` the states behind them come as a second result, fp32.
    Both states take part in the backward pass; second derivatives raise.

    Sequences are cut into chunks of 64 rows, ``T // 64 + N + 2`` of them at the most, however many are empty.  For each chunk and value head of 128 x 128 the call takes
    34 KB, with a graph 130 KB that it keeps beside its inputs for the backward pass, which takes another 64 KB while it runs (2.1 and 1 KB a row in long sequences; 1024
    sequences of 16 rows with 32 heads 5.5 and 2.7 GB).

    The lengths of a batch decide the order of fp32 sums: a sequence's results depend on its neighbours' lengths in their last bits.  Outputs and ``v``'s gradient are the
    exact ones rounded, but for one in some hundred; the gradients of q, k and a read the states between chunks as bf16 (off by 2.0e-3, 2.0e-3 and 1.8e-3 of their 2-norm
    where bf16 results are off by 1.7e-3).  States are off by some 3e-6.  What is not finite in a row's k, v, a or b reaches the rows of its own half chunk (32 rows)
    before it, too, and with a graph every gradient of its sequence; it stays out of other sequences."""
    out = _lib.host().gated_delta_rule(q, k, v, a, b, a_log, dt_bias, cu_seqlens, scale, bool(l2_norm), initial_state, bool(return_final_state))
    return tuple(out) if return_final_state else out[0]


@torch.compiler.disable
def gated_delta_step(q, k, v, a, b, a_log, dt_bias, state, *, scale=None, l2_norm: bool = True):
    """The next token of B requests: q, k (B, Hk, Dk), v (B, Hv, Dv), a, b (B, Hv) -> (B, Hv, Dv); ``state`` (B, Hv, Dk, Dv) fp32 is
    updated in place (a slice of a larger pool of requests will do).  No backward pass."""
    return _lib.host().gated_delta_step(q, k, v, a, b, a_log, dt_bias, state, scale, bool(l2_norm))


def _taps(weight):
    return weight.squeeze(1) if weight.dim() == 3 and weight.shape[1] == 1 else weight


def _silu(activation):
    if activation not in ("silu", "swish", None):
        raise ValueError(f"activation must be 'silu' or None, not {activation!r}")
    return activation is not None


@torch.compiler.disable
def short_conv(x, weight, bias, cu_seqlens, *, activation="silu", initial_state=None, return_final_state: bool = False):
    """x (T, channels) bf16 view, weight (channels, width) or (channels, 1, width), width 2 to 4, bias (channels,) or None -> (T, channels).

    Row t of a sequence sees the ``width - 1`` rows before it in the same sequence; before its first row lie ``initial_state`` (N, channels, width - 1) bf16, or
    zeros.  ``return_final_state`` adds each sequence's last ``width - 1`` inputs.  The states take no part in the backward pass; second derivatives raise.
    Rows behind the last sequence give zeros."""
    out = _lib.host().short_conv(x, _taps(weight), bias, cu_seqlens, _silu(activation), initial_state, bool(return_final_state))
    return tuple(out) if return_final_state else out[0]


@torch.compiler.disable
def short_conv_step(x, state, weight, bias=None, *, activation="silu"):
    """The next token of B requests: x (B, channels) -> (B, channels); ``state`` (B, channels, width - 1) bf16 moves on in place.  No backward pass."""
    return _lib.host().short_conv_step(x, state, _taps(weight), bias, _silu(activation))
