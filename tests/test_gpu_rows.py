"""Short convolution, gated norm and residual norm against their definitions in 64 bits (oracle/delta_ref.py).

Tolerances: the kernels compute in fp32 from exact inputs, so a bf16 result is off by its own rounding, at most 2^-8 of it, and by fp32 errors of the
terms it is a sum of: |err| <= 2^-8 |want| + 2^-16 (largest |want|).  The residual norm's backward reads x' as it is stored; where that is bf16, x' / |x'| carries 2^-8 of
its own into dw and one term of dx, dy: held to 2 * 2^-8 of the result's 2-norm instead.  fp32 results: 2^-18 of the 2-norm (sums of up to 2^13 terms)."""
import pytest
import torch

import vlm_training_amd as V
from oracle import delta_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _log(msg):
    print(f"[rows] {msg}", flush=True)


def cu_of(lens, dtype=torch.int32):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=dtype, device=DEV)


def close(got, want, name, wide=False):
    got, want = got.detach(), want.detach().double()
    f32, got = got.dtype == F32, got.double().cpu()
    assert got.shape == want.shape, name
    err = (got - want).abs()
    if f32 or wide:
        assert float(err.norm()) <= (2.0 ** -18 if f32 and not wide else 2.0 ** -7) * float(want.norm()) + 1e-30, (name, float(err.norm() / want.norm()))
    else:
        assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -16 * want.abs().max() + 1e-30).all(), (name, float((err / want.abs().max()).max()))


def leaves(d, where):
    return {n: (t.double() if where == "cpu" else t.to(DEV)).requires_grad_(True) if t is not None else None for n, t in d.items()}


@pytest.mark.parametrize("lens,C,W,bias,dtype,act", [
    ([1], 8, 4, False, BF, "silu"), ([2, 0, 1, 3], 24, 4, True, BF, "silu"), ([40, 1, 1, 1, 90], 264, 3, True, F32, None), ([500], 64, 2, False, F32, "silu"),
    ([1] * 70 + [30], 72, 4, True, BF, "silu"), ([300, 0, 0, 17], 2056, 4, False, BF, None),
])
def test_short_conv(lens, C, W, bias, dtype, act):
    _log(f"conv {lens[:5]} C {C} W {W}")
    g, T = torch.Generator().manual_seed(C + W), sum(lens)
    x = {"x": torch.randn(T + 5, C, generator=g).to(BF), "w": torch.randn(C, W, generator=g).to(dtype), "b": torch.randn(C, generator=g).to(dtype) if bias else None}
    dy, first = torch.randn(T + 5, C, generator=g).to(BF), torch.randn(len(lens), C, W - 1, generator=g).to(BF)
    for start in (None, first):
        c, d = leaves(x, "cpu"), leaves(x, DEV)
        want, last = R.short_conv(c["x"][:T], c["w"], c["b"], lens, start.double() if start is not None else None, act is not None)
        want.backward(dy[:T].double())
        got, state = V.short_conv(d["x"], d["w"].unsqueeze(1), d["b"], cu_of(lens), activation=act, initial_state=start.to(DEV) if start is not None else None,
                                  return_final_state=True)
        got.backward(dy.to(DEV))
        close(got[:T], want, "y")
        assert torch.equal(state.cpu().double(), last.detach()) and not got[T:].any() and not d["x"].grad[T:].any()
        close(d["x"].grad[:T], c["x"].grad[:T], "dx")
        close(d["w"].grad, c["w"].grad, "dw")
        if bias:
            close(d["b"].grad, c["b"].grad, "db")


def test_short_conv_of_views_and_its_steps():
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(50, 100, generator=g).to(BF).to(DEV)
    w = torch.randn(40, 4, generator=g).to(BF).to(DEV)
    want = V.short_conv(wide[:, 8:48].contiguous(), w, None, cu_of([30, 20]))
    assert torch.equal(V.short_conv(wide[:, 8:48], w, None, cu_of([30, 20], torch.int64)), want)              # 200-byte rows: copied
    assert torch.equal(V.short_conv(wide.t().contiguous().t()[:, 8:48], w, None, cu_of([30, 20])), want)
    x = wide[:, 8:48].contiguous()
    _, state = V.short_conv(x[:25], w, None, cu_of([25]), return_final_state=True)
    pool = torch.full((3, 1, 40, 3), 9.0, dtype=BF, device=DEV)
    pool[1] = state
    for t in range(25, 30):
        assert torch.equal(V.short_conv_step(x[t:t + 1], pool[1], w), want[t:t + 1])
    assert torch.equal(pool[1, 0], x[27:30].t()) and (pool[0] == 9).all() and (pool[2] == 9).all()


@pytest.mark.parametrize("T,H,D,dtype,offset", [(1, 1, 8, BF, False), (13, 3, 72, F32, True), (300, 5, 128, BF, False), (2000, 32, 64, BF, False), (7, 2, 512, F32, False)])
def test_gated_rms_norm(T, H, D, dtype, offset):
    _log(f"gated norm {T} {H} {D}")
    g = torch.Generator().manual_seed(T + D)
    x = {"x": torch.randn(T, H, D, generator=g).to(BF), "z": (2 * torch.randn(T, H, D, generator=g)).to(BF), "w": torch.randn(D, generator=g).to(dtype)}
    dy = torch.randn(T, H, D, generator=g).to(BF)
    c, d = leaves(x, "cpu"), leaves(x, DEV)
    want = R.gated_rms_norm(*c.values(), offset=offset)
    want.backward(dy.double())
    got = V.gated_rms_norm(*d.values(), offset=offset)
    got.backward(dy.to(DEV))
    close(got, want, "y")
    for n in x:
        close(d[n].grad, c[n].grad, n)


@pytest.mark.parametrize("C", [24, 264])
def test_what_is_not_finite_stays_in_its_sequence(C):
    lens, T = [13, 5, 0, 60, 1, 40], 119
    x, dy = torch.randn(T + 30, C, device=DEV).to(BF), torch.randn(T + 30, C, device=DEV).to(BF)
    w, b, cu = torch.randn(C, 4, device=DEV).to(BF), torch.randn(C, device=DEV).to(BF), cu_of(lens)

    def run():
        leaf = x.clone().requires_grad_(True)
        y = V.short_conv(leaf, w, b, cu)
        return y.detach(), torch.autograd.grad(y, leaf, dy)[0]

    want = run()
    for lo, hi in ((T, T + 30), (18, 78), (0, 13)):      # rows behind the last sequence, then two whole sequences
        x[lo:hi] = float("nan")
        dy[lo:hi] = float("inf")
        for got, ref in zip(run(), want):
            keep = torch.ones(T + 30, dtype=torch.bool, device=DEV)
            keep[18:78] &= hi > T
            keep[:13] &= lo > 0
            assert torch.equal(got[keep], ref[keep])
    z = torch.randn(9, 3, 64, device=DEV).to(BF)
    z[4, 1] = float("nan")
    y = V.gated_rms_norm(z, torch.ones_like(z), torch.ones(64, device=DEV))
    assert torch.isfinite(y).all(-1).logical_not().nonzero().tolist() == [[4, 1]]


def test_gated_rms_norm_reads_views_in_place():
    x = torch.randn(20, 3, 2 * 64, device=DEV).to(BF)
    w = torch.ones(64, device=DEV)
    assert torch.equal(V.gated_rms_norm(x[..., :64], x[..., 64:], w), V.gated_rms_norm(x[..., :64].contiguous(), x[..., 64:].contiguous(), w))
    odd = torch.zeros(20 * 3 * 64 + 1, device=DEV, dtype=BF)[1:].view(20, 3, 64).copy_(x[..., :64])
    assert torch.equal(V.gated_rms_norm(odd, x[..., 64:], w), V.gated_rms_norm(x[..., :64], x[..., 64:], w))


def test_norms_of_zero_rows_and_large_ones():
    x = torch.zeros(4, 2, 64, device=DEV, dtype=BF)
    x[1] = 3e18                                          # squares within fp32
    y = V.gated_rms_norm(x, torch.ones_like(x), torch.ones(64, device=DEV))
    assert not y[0].any() and torch.allclose(y[1].float(), torch.sigmoid(torch.tensor(1.0)).to(DEV).expand(2, 64), rtol=2.0 ** -8)
    new, h = V.residual_rms_norm(torch.zeros(3, 64, device=DEV, dtype=BF), torch.zeros(3, 64, device=DEV, dtype=BF), torch.ones(64, device=DEV))
    assert not new.any() and not h.any()


@pytest.mark.parametrize("post,gate,scale", [(p, g, s) for p in (0, 1) for g in (0, 1) for s in (0, 1)])
@pytest.mark.parametrize("T,C,stream,dtype", [(1, 8, BF, BF), (37, 520, F32, F32), (130, 1000, BF, F32), (5, 2056, F32, BF), (3, 8192, BF, BF)])
def test_residual_rms_norm(T, C, stream, dtype, post, gate, scale):
    _log(f"residual norm {T} {C} {post}{gate}{scale}")
    g = torch.Generator().manual_seed(T + C)
    rn = lambda *s: torch.randn(*s, generator=g)
    x = {"x": (2 * rn(T, C)).to(stream), "y": rn(T, C).to(BF), "w": rn(C).to(dtype), "post": rn(C).to(dtype) if post else None,
         "gate": rn(T, C).to(BF) if gate else None, "scale": rn(C).to(dtype) if scale else None}
    grads = rn(T, C).to(stream), rn(T, C).to(BF)
    c, d = leaves(x, "cpu"), leaves(x, DEV)
    want = R.residual_rms_norm(*c.values(), offset=bool(post))
    torch.autograd.backward(want, [t.double() for t in grads])
    got = V.residual_rms_norm(d["x"], d["y"], d["w"], post_weight=d["post"], gate=d["gate"], scale=d["scale"], offset=bool(post))
    torch.autograd.backward(got, [t.to(DEV) for t in grads])
    close(got[0], want[0], "x'")
    close(got[1], want[1], "h")
    for n in x:
        if x[n] is not None:
            close(d[n].grad, c[n].grad, n, wide=stream == BF)


def test_residual_rms_norm_with_one_gradient_and_more_dimensions():
    g = torch.Generator().manual_seed(4)
    x, y, w = torch.randn(2, 5, 64, generator=g).to(DEV).to(BF), torch.randn(2, 5, 64, generator=g).to(DEV).to(BF), torch.randn(64, generator=g).to(DEV)
    dy = torch.randn(2, 5, 64, generator=g).to(DEV).to(BF)
    for which in (0, 1):
        a = [t.clone().requires_grad_(True) for t in (x, y, w)]
        b = [t.cpu().double().requires_grad_(True) for t in (x, y, w)]
        V.residual_rms_norm(*a, scale=0.5)[which].backward(dy)
        R.residual_rms_norm(*b, scale=0.5)[which].backward(dy.cpu().double())
        for p, q, n in zip(a, b, "xyw"):
            if q.grad is not None:
                close(p.grad, q.grad, (which, n), wide=True)
        if which == 0:
            assert not a[2].grad.any()
    assert a[0].grad.data_ptr() != a[1].grad.data_ptr()


def test_captured_and_replayed():
    g = torch.Generator().manual_seed(5)
    x = torch.randn(200, 64, generator=g).to(BF).to(DEV).requires_grad_(True)
    w = torch.randn(64, 4, generator=g).to(BF).to(DEV).requires_grad_(True)
    n = torch.ones(64, device=DEV).requires_grad_(True)
    dy, cu = torch.randn(200, 64, generator=g).to(BF).to(DEV), cu_of([150, 50])

    def step():
        y = V.short_conv(x, w, None, cu)
        y = V.gated_rms_norm(y.unsqueeze(1), x.unsqueeze(1), n).squeeze(1)
        new, h = V.residual_rms_norm(x, y, n)
        return [new.detach(), h.detach(), *torch.autograd.grad([new, h], [x, w, n], [dy, dy])]

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for replay in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        other = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(got, want, other)), replay


def test_empty_batches():
    x = torch.empty(0, 64, dtype=BF, device=DEV, requires_grad=True)
    w = torch.ones(64, 4, device=DEV, requires_grad=True)
    y, s = V.short_conv(x, w, None, cu_of([0]), return_final_state=True)
    y.sum().backward()
    assert y.shape == (0, 64) and not s.any() and not w.grad.any()
    n = torch.ones(64, device=DEV, requires_grad=True)
    V.gated_rms_norm(x.view(0, 1, 64), x.view(0, 1, 64), n).sum().backward()
    assert not n.grad.any()
    new, h = V.residual_rms_norm(x, x, n)
    (new.sum() + h.sum()).backward()
    assert new.shape == (0, 64) and not n.grad.any()
    assert V.short_conv_step(x.detach(), torch.empty(0, 64, 3, dtype=BF, device=DEV), w.detach()).shape == (0, 64)


def test_refusals():
    x, cu = torch.zeros(10, 64, dtype=BF, device=DEV), cu_of([10])
    w, s = torch.zeros(64, 4, device=DEV), torch.zeros(10, 64, 3, dtype=BF, device=DEV)
    for bad in ((x.float(), w, None), (x, w[:32], None), (x, w, w[:3, 0]), (x, w.half(), None), (x[0], w, None)):
        with pytest.raises(ValueError):
            V.short_conv(*bad, cu)
    with pytest.raises(ValueError, match="activation"):
        V.short_conv(x, w, None, cu, activation="relu")
    with pytest.raises(ValueError, match="detach"):
        V.short_conv(x, w, None, cu, initial_state=s[:1].clone().requires_grad_(True))
    with pytest.raises(ValueError):
        V.short_conv(x, w, None, cu, initial_state=s[:1].float())
    with pytest.raises(RuntimeError, match="width"):
        V.short_conv(x, torch.zeros(64, 5, device=DEV), None, cu)
    with pytest.raises(RuntimeError, match="channels"):
        V.short_conv(x[:, :60].contiguous(), w[:60], None, cu)
    with pytest.raises(ValueError, match="in place"):
        V.short_conv_step(x, s[:1].expand(10, 64, 3), w)
    with pytest.raises(ValueError, match="backward"):
        V.short_conv_step(x, s, w.clone().requires_grad_(True))
    r = x.view(10, 1, 64)
    for bad in ((r.float(), r, w[:, 0]), (r, r[:5], w[:, 0]), (r, r, w[:32, 0]), (r, r, w[:, 0].half()), (x, x, w[:, 0])):
        with pytest.raises(ValueError):
            V.gated_rms_norm(*bad)
    with pytest.raises(RuntimeError, match="up to 512"):
        V.gated_rms_norm(torch.zeros(1, 1, 520, dtype=BF, device=DEV), torch.zeros(1, 1, 520, dtype=BF, device=DEV), torch.zeros(520, device=DEV))
    for bad in ((x.half(), x, w[:, 0]), (x, x.float(), w[:, 0]), (x, x[:5], w[:, 0]), (x, x, w[:3, 0])):
        with pytest.raises(ValueError):
            V.residual_rms_norm(*bad)
    with pytest.raises(ValueError):
        V.residual_rms_norm(x, x, w[:, 0], gate=x.float())
    with pytest.raises(RuntimeError, match="up to 8192"):
        V.residual_rms_norm(torch.zeros(1, 8200, dtype=BF, device=DEV), torch.zeros(1, 8200, dtype=BF, device=DEV), torch.zeros(8200, device=DEV))
    with pytest.raises(RuntimeError, match="GPU only"):
        V.residual_rms_norm(x.cpu(), x.cpu(), w[:, 0].cpu())
