"""Elements past 2^31: the last rows of tensors that long equal the same rows computed alone."""
import pytest
import torch

import vlm_training_amd as V

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


@pytest.fixture(autouse=True)
def _free():
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GB of free device memory")
    yield
    torch.cuda.empty_cache()


def rows(n, *shape):
    """n rows that repeat after 4099 of them, so that they are made fast and no two neighbouring blocks are equal"""
    g = torch.Generator(device=DEV).manual_seed(n)
    block = torch.randn(4099, *shape, device=DEV, generator=g).to(BF)
    return block.repeat(n // 4099 + 1, *([1] * len(shape)))[:n]


def test_short_convolution():
    T, C = 263_000, 8192                                 # 2.15e9 elements
    x, dy = rows(T, C).requires_grad_(True), rows(T, C)
    w, bias = torch.randn(C, 4, device=DEV).to(BF), torch.randn(C, device=DEV).to(BF)
    cut = T - 700
    y = V.short_conv(x, w, bias, torch.tensor([0, cut, T], device=DEV, dtype=torch.int32))
    dx, = torch.autograd.grad(y, x, dy)
    tail = x.detach()[cut:].clone().requires_grad_(True)
    y2 = V.short_conv(tail, w, bias, torch.tensor([0, 700], device=DEV, dtype=torch.int32))
    dx2, = torch.autograd.grad(y2, tail, dy[cut:])
    assert torch.equal(y[cut:], y2) and torch.equal(dx[cut:], dx2)


def test_norms():
    T, H, D = 262_500, 64, 128
    x, z, dy = rows(T, H, D).requires_grad_(True), rows(T, H, D), rows(T, H, D)
    w = torch.randn(D, device=DEV)
    y = V.gated_rms_norm(x, z, w)
    dx, = torch.autograd.grad(y, x, dy)
    tail = x.detach()[-50:].clone().requires_grad_(True)
    y2 = V.gated_rms_norm(tail, z[-50:], w)
    assert torch.equal(y[-50:], y2) and torch.equal(dx[-50:], torch.autograd.grad(y2, tail, dy[-50:])[0])
    x, z, dy = (t.detach().reshape(-1, 8192) for t in (x, z, dy))
    x.requires_grad_(True)
    w = w.repeat(64)
    new, h = V.residual_rms_norm(x, z, w)
    dx, = torch.autograd.grad([new, h], x, [dy, dy])
    tail = x.detach()[-50:].clone().requires_grad_(True)
    new2, h2 = V.residual_rms_norm(tail, z[-50:], w)
    assert torch.equal(new[-50:], new2) and torch.equal(h[-50:], h2) and torch.equal(dx[-50:], torch.autograd.grad([new2, h2], tail, [dy[-50:], dy[-50:]])[0])


def test_gated_delta_rule():
    T, hk, hv, d = 530_000, 4, 32, 128                   # v, the output and their gradients 2.17e9 elements, the workspaces 1.1e9 bytes a head
    tail = 40_000
    q, k, v, dout = rows(T, hk, d), rows(T, hk, d), rows(T, hv, d), rows(T, hv, d)
    a, b = rows(T, hv), rows(T, hv)
    a_log, dt = torch.zeros(hv, device=DEV, dtype=BF), torch.zeros(hv, device=DEV, dtype=BF)
    lens = [T - tail] + [tail // 20] * 20
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)
    leaves = [t.requires_grad_(True) for t in (q, k, v, a, b)]
    o = V.gated_delta_rule(*leaves, a_log, dt, cu)
    got = [o.detach()[-tail:].clone()] + [g[-tail:].clone() for g in torch.autograd.grad(o, leaves, dout)]
    del o
    part = [torch.cat([t.detach()[:1], t.detach()[-tail:]]).requires_grad_(True) for t in leaves]
    cu2 = torch.tensor([0, 1] + [tail // 20] * 20, device=DEV).cumsum(0).to(torch.int32)
    o2 = V.gated_delta_rule(*part, a_log, dt, cu2)
    want = [o2.detach()[1:]] + [g[1:] for g in torch.autograd.grad(o2, part, torch.cat([dout[:1], dout[-tail:]]))]
    # The lengths decide how the walks are split, and with it the order of fp32 sums: the two runs are equal up to twice what each may be off from the definition
    # (4.6e-3 of the output's 2-norm, 1e-2 of a gradient's: the triangle inequality).
    for i, (x, y) in enumerate(zip(got, want)):
        assert float((x.float() - y.float()).norm()) <= 2 * (4.6e-3 if i == 0 else 1e-2) * float(y.float().norm())


def test_single_tokens():
    B, hk, hv, d = 4200, 16, 32, 128                     # 2.2e9 elements of state
    state = torch.empty(B, hv, d, d, device=DEV).normal_()
    conv = rows(B, 8192, 3)
    x = [rows(B, n, d) for n in (hk, hk, hv)] + [rows(B, hv), rows(B, hv)]
    a_log, dt = torch.zeros(hv, device=DEV, dtype=BF), torch.zeros(hv, device=DEV, dtype=BF)
    last = state[-9:].clone()
    with torch.no_grad():
        o = V.gated_delta_step(*x, a_log, dt, state)
        o2 = V.gated_delta_step(*(t[-9:] for t in x), a_log, dt, last)
    assert torch.equal(o[-9:], o2) and torch.equal(state[-9:], last)
    w, row, last = torch.randn(8192, 4, device=DEV).to(BF), rows(B, 8192), conv[-9:].clone()
    with torch.no_grad():
        y = V.short_conv_step(row, conv, w)
        assert torch.equal(y[-9:], V.short_conv_step(row[-9:].contiguous(), last, w)) and torch.equal(conv[-9:], last)
