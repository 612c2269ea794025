"""A gated-delta-rule layer between residual additions, as the hybrid stack runs it, against the same built from the 64-bit definitions."""
from types import SimpleNamespace

import pytest
import torch

import vlm_training_amd as V
from oracle import delta_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
CFG = SimpleNamespace(hidden_size=256, linear_num_key_heads=2, linear_num_value_heads=8, linear_key_head_dim=64, linear_value_head_dim=64, linear_conv_kernel_dim=4,
                      rms_norm_eps=1e-6)


def build(seed=0):
    torch.manual_seed(seed)
    layer, before, after = V.GatedDeltaNet(CFG), torch.randn(256) * 0.1 + 1, torch.randn(256) * 0.1 + 1
    for p in layer.parameters():
        p.data = p.data.bfloat16()
    return layer, before.bfloat16(), after.bfloat16()


def oracle(layer, before, after, x, y, lens):
    """residual norm -> layer -> residual norm on (T, hidden) in double."""
    p = {n: t for n, t in layer.items()}
    new, h = R.residual_rms_norm(x, y, before)
    mixed, _ = R.short_conv(h @ p["in_proj_qkv.weight"].t(), p["conv1d.weight"].squeeze(1), None, lens)
    q, k, v = mixed.split((128, 128, 512), 1)
    heads = lambda t: t.unflatten(1, (-1, 64))
    o, _ = R.gated_delta_rule(heads(q), heads(k), heads(v), h @ p["in_proj_a.weight"].t(), h @ p["in_proj_b.weight"].t(), p["A_log"], p["dt_bias"], lens)
    o = R.gated_rms_norm(o, heads(h @ p["in_proj_z.weight"].t()), p["norm.weight"])
    return R.residual_rms_norm(new, o.flatten(1) @ p["out_proj.weight"].t(), after)


@pytest.mark.parametrize("lens", [[50, 1, 80], [2200]])      # (the longer one takes the shared projections)
def test_block_forward_and_every_gradient(lens):
    """bf16 hand-overs between the parts (projection, convolution, rule, norm, projection, norm: seven deep, each 2^-8 / sqrt(3) of the values in the mean
    square) add up to 6e-3 of the forward; the backward passes as many again: 1.2e-2, twice that for the smallest parameters' sums."""
    layer, before, after = build()
    T, g = sum(lens), torch.Generator().manual_seed(1)
    x, y = torch.randn(T, 256, generator=g).bfloat16(), torch.randn(T, 256, generator=g).bfloat16()
    grads = [torch.randn(T, 256, generator=g).bfloat16() for _ in range(2)]
    want_p = {n: t.detach().double().requires_grad_(True) for n, t in layer.named_parameters()}
    wx, wb = x.double().requires_grad_(True), before.double().requires_grad_(True)
    want = oracle(want_p, wb, after.double(), wx, y.double(), lens)
    torch.autograd.backward(want, [t.double() for t in grads])
    layer = layer.to(DEV)
    gx, gb = x.to(DEV).requires_grad_(True), before.to(DEV).requires_grad_(True)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=DEV)
    new, h = V.residual_rms_norm(gx, y.to(DEV), gb)
    out = V.residual_rms_norm(new, layer(h.unsqueeze(0), cu).squeeze(0), after.to(DEV))
    torch.autograd.backward(out, [t.to(DEV) for t in grads])
    off = lambda a, b: float((a.detach().double().cpu() - b.detach()).norm() / b.detach().norm())
    for a, b in zip(out, want):
        assert off(a, b) <= 6e-3, off(a, b)
    assert off(gx.grad, wx.grad) <= 1.2e-2 and off(gb.grad, wb.grad) <= 2.4e-2
    for n, p in layer.named_parameters():
        assert off(p.grad, want_p[n].grad) <= (2.4e-2 if p.numel() < 4096 else 1.2e-2), (n, off(p.grad, want_p[n].grad))


def test_prefill_in_two_parts_and_steps_agree_with_one_pass():
    """The same rows in one packed pass, in two with the state between them, and token by token: outputs to the layer's own rounding."""
    layer, _, _ = build(2)
    layer = layer.to(DEV)
    x = torch.randn(1, 120, 256, generator=torch.Generator().manual_seed(3)).bfloat16().to(DEV)
    cu = lambda *e: torch.tensor(e, dtype=torch.int32, device=DEV)
    with torch.no_grad():
        whole = layer(x, cu(0, 60, 120)).squeeze(0)
        rows = torch.cat([torch.arange(0, 40), torch.arange(60, 100)])
        first, state = layer(x[:, rows], cu(0, 40, 80), return_state=True)
        rows2 = torch.cat([torch.arange(40, 55), torch.arange(100, 115)])
        second, state = layer(x[:, rows2], cu(0, 15, 30), state=state, return_state=True)
        off = lambda a, b: float((a.double() - b.double()).norm() / b.double().norm())
        assert off(first.squeeze(0), whole[rows]) <= 6e-3 and off(second.squeeze(0), whole[rows2]) <= 6e-3
        for t in range(5):
            at = torch.tensor([55 + t, 115 + t])
            assert off(layer.step(x[0, at], state), whole[at]) <= 6e-3


def test_layer_under_autocast_and_with_fp32_parameters():
    """fp32 master weights under bf16 autocast, as the trainer holds them."""
    torch.manual_seed(4)
    layer = V.GatedDeltaNet(CFG).to(DEV)
    x = torch.randn(1, 90, 256, device=DEV, requires_grad=True)
    cu = torch.tensor([0, 90], dtype=torch.int32, device=DEV)
    with torch.autocast("cuda", torch.bfloat16):
        out = layer(x, cu)
    out.float().sum().backward()
    assert all(p.grad is not None and p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all() for p in layer.parameters())
    same = V.GatedDeltaNet(CFG).to(DEV)
    same.load_state_dict(layer.state_dict())
    with torch.no_grad():
        want = same.bfloat16()(x.bfloat16(), cu)
    assert float((out.float() - want.float()).norm() / want.float().norm()) <= 2e-2
