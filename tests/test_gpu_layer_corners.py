"""Short convolution, gated norm and residual norm where their formulas are easily lost: gates at the type's lowest value, large pre-activations, gradients of a
bf16 residual stream, second derivatives.  Tolerances as in test_gpu_rows.py: a bf16 result's own rounding, 2^-8 of it, and 2^-16 of the largest."""
import ctypes

import pytest
import torch

import vlm_training_amd as V
from oracle import delta_ref as R
from tests.test_gpu_rows import close, cu_of, leaves
from vlm_training_amd import _lib

pytestmark = pytest.mark.gpu
DEV, BF, F32 = "cuda", torch.bfloat16, torch.float32


def _log(msg):
    print(f"[corners] {msg}", flush=True)


def test_gated_norm_with_gates_at_the_lowest_value():
    """silu of the lowest bf16 is -0 (its sigmoid is 0): so are the row's outputs there, and its gradients."""
    low = torch.finfo(BF).min
    g = torch.Generator().manual_seed(1)
    x = {"x": torch.randn(6, 3, 64, generator=g).to(BF), "z": torch.randn(6, 3, 64, generator=g).to(BF), "w": 1 + torch.rand(64, generator=g)}
    x["z"][1] = low
    x["z"][2, :, ::2] = low
    x["z"][3] = torch.tensor([-1e30, -3e4, -200., -100., -88., -60., 60., 1e4]).repeat(8).to(BF)
    dy = torch.randn(6, 3, 64, generator=g).to(BF)
    dy[3] *= 2.0 ** -12                                  # (its largest gate is 1e4: the others' rows set the tolerance)
    c, d = leaves(x, "cpu"), leaves(x, DEV)
    want = R.gated_rms_norm(*c.values())
    want.backward(dy.double())
    got = V.gated_rms_norm(*d.values())
    got.backward(dy.to(DEV))
    assert torch.isfinite(got).all() and not got[1].any()
    close(got, want, "y")
    for n in x:
        assert torch.isfinite(d[n].grad).all(), n
        close(d[n].grad, c[n].grad, n)


@pytest.mark.parametrize("W", [2, 3, 4])
def test_convolution_with_large_values(W):
    """silu'(z) is 1 for every large z and 0 for every low one."""
    g = torch.Generator().manual_seed(W)
    T, C = 80, 24
    size = 2.0 ** torch.linspace(0, 40, T)[:, None]
    x = (torch.randn(T, C, generator=g).sign() * size * (1 + torch.rand(T, C, generator=g))).to(BF)
    x[-1] = torch.finfo(BF).min
    w = torch.zeros(C, W)
    w[:, W - 1] = 1.0                                    # z = x
    dy = torch.randn(T, C, generator=g).to(BF)
    args = {"x": x, "w": w, "b": torch.zeros(C)}
    c, d = leaves(args, "cpu"), leaves(args, DEV)
    want, _ = R.short_conv(c["x"], c["w"], c["b"], [T])
    want.backward(dy.double())
    got = V.short_conv(d["x"], d["w"], d["b"], cu_of([T]))
    got.backward(dy.to(DEV))
    # (below -88.7 e^-z passes fp32's range and z sigmoid(z) becomes 0: off by 89 e^-88.7 = 2.7e-37 at the most)
    assert ((got.cpu().double() - want.detach()).abs() <= 2.0 ** -8 * want.detach().abs() + 3e-37).all() and not got[-1].any()
    close(d["x"].grad, c["x"].grad, "dx")
    close(d["b"].grad, c["b"].grad, "db")


@pytest.mark.parametrize("post,gate,scale", [(p, g, s) for p in (0, 1) for g in (0, 1) for s in (0, 1)])
@pytest.mark.parametrize("T,C", [(1, 8), (130, 1000), (700, 264), (5, 2056), (3, 8192)])
def test_gradients_of_a_bf16_stream_are_those_of_the_unrounded_one(T, C, post, gate, scale):
    """The forward's norm reads x' before it is rounded, and its gradient is taken there."""
    _log(f"residual norm {T} {C} {post}{gate}{scale}")
    g = torch.Generator().manual_seed(T + C + 1)
    rn = lambda *s: torch.randn(*s, generator=g)
    x = {"x": (2 * rn(T, C)).to(BF), "y": rn(T, C).to(BF), "w": rn(C), "post": rn(C) if post else None, "gate": rn(T, C).to(BF) if gate else None,
         "scale": rn(C) if scale else None}
    grads = rn(T, C).to(BF), rn(T, C).to(BF)
    c, d = leaves(x, "cpu"), leaves(x, DEV)
    torch.autograd.backward(R.residual_rms_norm(*c.values(), offset=bool(gate)), [t.double() for t in grads])
    got = V.residual_rms_norm(d["x"], d["y"], d["w"], post_weight=d["post"], gate=d["gate"], scale=d["scale"], offset=bool(gate))
    torch.autograd.backward(got, [t.to(DEV) for t in grads])
    for n in x:
        if x[n] is not None:
            close(d[n].grad, c[n].grad, n)


def test_gradients_through_the_c_entry_with_a_rounded_stream():
    """DSA_STREAM_BF16 takes x' as a bf16 stream holds it: its rounding, 2^-8 of a value at the most, is in dw and in one term of dx (2 * 2^-8 of the 2-norm)."""
    T, C = 130, 264
    g = torch.Generator().manual_seed(5)
    rn = lambda *s: torch.randn(*s, generator=g)
    x, y, w, dxn, dh = (2 * rn(T, C)).to(BF), rn(T, C).to(BF), rn(C), rn(T, C).to(BF), rn(T, C).to(BF)
    c = {n: t.double().requires_grad_(True) for n, t in (("x", x), ("y", y), ("w", w))}
    torch.autograd.backward(R.residual_rms_norm(c["x"], c["y"], c["w"]), [dxn.double(), dh.double()])
    d = [t.to(DEV) for t in (x, y, w, dxn, dh)]
    xn, h, dx, dy = (torch.empty(T, C, dtype=BF, device=DEV) for _ in range(4))
    rstd, dw = torch.empty(T, device=DEV), torch.empty(C, device=DEV)
    lib, p = _lib.load(), lambda t: ctypes.c_void_p(t.data_ptr())
    n = lib.dsa_residual_norm_bwd_workspace_bytes(T, C)
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.dsa_residual_norm_fwd(p(d[0]), 0, p(d[1]), None, p(d[2]), 1, None, 0, None, 0, 1e-6, 0.0, T, C, p(xn), p(h), p(rstd), None, stream) == 0
    for kind, wide in ((0, True), (2, False)):
        assert lib.dsa_residual_norm_bwd(p(d[3]), p(d[4]), p(xn if kind == 0 else d[0]), kind, p(d[1]), None, p(d[2]), 1, None, 0, None, 0, 0.0, T, C, p(rstd), None, p(dx),
                                         p(dy), None, p(dw), None, None, p(ws), n, stream) == 0
        torch.cuda.synchronize()
        for name, got, want in (("dx", dx, c["x"].grad), ("dy", dy, c["y"].grad), ("dw", dw, c["w"].grad)):
            close(got, want, (kind, name), wide=wide)


def test_stream_kinds_that_are_none_are_refused():
    lib = _lib.load()
    n = lib.dsa_residual_norm_bwd_workspace_bytes(4, 64)
    bwd = lambda kind, y: lib.dsa_residual_norm_bwd(16, 16, 16, kind, y, None, 16, 0, None, 0, None, 0, 0.0, 4, 64, 16, None, 16, 16, None, 16, None, None, 16, n - 1, None)
    assert bwd(3, 16) == -1 and bwd(-1, 16) == -1 and bwd(2, None) == -1 and bwd(2, 16) == -3 and bwd(0, None) == -3
    fwd = lambda kind, h: lib.dsa_residual_norm_fwd(16, kind, 16, None, 16, 0, None, 0, None, 0, 1e-6, 0.0, 4, 64, 16, h, None, None, None)
    assert fwd(2, 16) == -1 and b"x_f32" in lib.dsa_last_error() and fwd(1, None) == -1 and b"null" in lib.dsa_last_error()


def test_second_derivatives_are_refused():
    """With create_graph the gradients are the same, and what would need their own derivatives raises - of an input, of a gradient that came in, or of everything at once -
    rather than leave that share out."""
    def leaf():
        return torch.randn(70, 64, device=DEV, generator=torch.Generator(DEV).manual_seed(3)).to(BF).requires_grad_(True)

    w4, n, cu = torch.randn(64, 4, device=DEV), torch.ones(64, device=DEV, requires_grad=True), cu_of([70])
    a, p = torch.zeros(70, 1, device=DEV), torch.zeros(1, device=DEV)
    calls = {"gated_delta_rule": lambda x: V.gated_delta_rule(*[x.unsqueeze(1)] * 3, a, a, p, p, cu).squeeze(1), "short_conv": lambda x: V.short_conv(x, w4, None, cu),
             "gated_rms_norm": lambda x: V.gated_rms_norm(x.unsqueeze(1), x.unsqueeze(1), n).squeeze(1), "residual_rms_norm": lambda x: V.residual_rms_norm(x, x, n)[1]}
    for name, call in calls.items():
        x, dy = leaf(), torch.randn(70, 64, device=DEV).to(BF)
        want, = torch.autograd.grad(call(x), x, dy)
        dy = dy.clone().requires_grad_(True)
        first, = torch.autograd.grad(call(x), x, dy, create_graph=True)
        assert torch.equal(first, want) and first.requires_grad, name
        penalty = first.float().square().sum() + x.float().square().sum() + dy.float().sum()
        for ask in (lambda: torch.autograd.grad(penalty, x, retain_graph=True), lambda: torch.autograd.grad(penalty, dy, retain_graph=True), lambda: penalty.backward()):
            with pytest.raises(NotImplementedError, match=name + ": second"):
                ask()
