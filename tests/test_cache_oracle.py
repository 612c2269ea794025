"""The 64-bit restatement of the paged cache against torch's own e4m3 and attention: runs without a GPU."""
import math

import torch

from oracle import cache_ref as R


def test_every_e4m3_value_is_kept():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    codes = codes[torch.isfinite(codes)]
    rows = torch.stack([codes, codes * 2.0 ** 20, codes * 2.0 ** -60])
    got, e = R.quantise(rows)
    assert e.tolist() == [0, 20, -60] and torch.equal(got, codes.expand(3, -1))


def test_rounding_is_torchs():
    x = torch.randn(64, 96, generator=torch.Generator().manual_seed(0)) * torch.logspace(-6, 6, 64)[:, None]
    x[3] = 0
    got, e = R.quantise(x)
    want = (x.double() * torch.exp2(-e.double())[:, None]).float().to(torch.float8_e4m3fn).double()
    assert torch.equal(got, want) and e[3] == -100
    top = x.double().abs().amax(-1) * torch.exp2(-e.double())
    live = top > 0
    assert (top <= 448).all() and (top[live] > 224).all()


def test_rows_that_are_not_finite():
    x = torch.ones(3, 16)
    x[0, 2], x[1, 3] = math.inf, math.nan
    got = R.stored(x, "e4m3")
    assert torch.isnan(got[:2]).all() and torch.equal(got[2], torch.ones(16, dtype=torch.float64))


def test_attention_is_torchs():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, h, 24, generator=g, dtype=torch.float64) for n, h in ((5, 6), (9, 2), (9, 2)))
    out, lse = R.attend(q, k, v, 0.3, [4, 5, 6, 7, 8])
    mask = torch.arange(9)[None] <= torch.arange(4, 9)[:, None]
    want = torch.nn.functional.scaled_dot_product_attention(q.transpose(0, 1), k.repeat_interleave(3, 1).transpose(0, 1), v.repeat_interleave(3, 1).transpose(0, 1),
                                                            attn_mask=mask, scale=0.3).transpose(0, 1)
    assert (out - want).abs().max() < 1e-13
    logits = torch.einsum("ihd,lhd->hil", q, k.repeat_interleave(3, 1)) * 0.3
    assert (lse - logits.masked_fill(~mask, -math.inf).logsumexp(-1)).abs().max() < 1e-13
    out, lse = R.attend(q, k, v, 0.3, [-2, -1, 0, 1, 2])
    assert (out[:2] == 0).all() and (lse[:, :2] == -math.inf).all() and torch.allclose(out[2], v[0].repeat_interleave(3, 0))
