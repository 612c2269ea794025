"""Gradients of the decay where they are differences of sums that cancel, what the products' low halves are there for, and bits past 2^31 elements.

Bounds.  A value kept as two bf16 is off by 2^-18 of itself, one bf16 by 2^-9.  A row's dG is a sum of three kinds of terms: pairs of rows inside the chunk (X and
Z, two bf16 each, from N and dR of two bf16 each, products without lo x lo: 2^-16 of every pair's absolute value, which itself counts with the absolute values
of the sums T R and T^T dN behind N and dR), products with the states S0 and dS1 at the chunk's borders (kept as one bf16: 2^-9, and N or dR beside them 2^-9 at the
most) and <dS1, S0> (both: 2^-8).  dg of a row sums dG from it on.  Everything is formed here in 64 bits from the definition."""
import pytest
import torch

import vlm_training_amd as V
from oracle import delta_ref as R
from tests.test_gpu_delta import DEV, GRAD, NAMES, cu_of, inputs

pytestmark = pytest.mark.gpu


def _log(msg):
    print(f"[heads] {msg}", flush=True)


def grads_of(x, lens):
    leaves = [x[n].to(DEV).requires_grad_(True) for n in NAMES]
    o = V.gated_delta_rule(*leaves, cu_of(lens))
    got = torch.autograd.grad(o, leaves, x["dout"].to(DEV))
    torch.cuda.synchronize()
    return o.detach().cpu(), {n: g.cpu() for n, g in zip(NAMES, got)}


@pytest.mark.parametrize("hv,d", [(4, 64), (6, 128)])
@pytest.mark.parametrize("change", ["large", "nan", "inf"])
def test_a_value_head_leaves_the_others_of_its_key_head_alone(hv, d, change):
    """The first head of each key head a million times as large, or not finite: every result of the others' own is the same to the bit."""
    _log(f"{change} first heads, {hv} heads of {d}")
    hk = 2
    first = [u for u in range(hv) if u % (hv // hk) == 0]
    rest = [u for u in range(hv) if u not in first]
    lens = [150, 70]
    x = inputs(220, hk, hv, d, d, seed=50 + hv, dtype=torch.float32)
    o, want = grads_of(x, lens)
    for n in ("v", "dout"):
        x[n] = x[n].clone()
        if change == "large":
            x[n][:, first] *= 2.0 ** 20
        else:
            x[n][5:, first] = float(change)
    o2, got = grads_of(x, lens)
    assert torch.equal(o2[:, rest], o[:, rest])
    for n in ("v", "a", "b"):
        assert torch.isfinite(want[n]).all()
        assert torch.equal(got[n][:, rest], want[n][:, rest]), n
    for n in ("a_log", "dt_bias"):
        assert torch.equal(got[n][rest], want[n][rest]), n


def decay_gradients(x, lens, scale=None):
    """Exact da, db, da_log, ddt_bias (in 64 bits, from the recurrence) and how far the kernels' may be off, all (T, Hv) per row."""
    T, hk, dk = x["q"].shape
    hv, dv = x["v"].shape[1:]
    scale = dk ** -0.5 if scale is None else scale
    q, k = (R.unit(x[n].double()).repeat_interleave(hv // hk, 1) for n in "qk")
    a, b = x["a"].double(), x["b"].double()
    rate = torch.exp(x["a_log"].double())
    z = a + x["dt_bias"].double()
    g = (-rate * torch.nn.functional.softplus(z, threshold=60)).requires_grad_(True)
    beta = torch.sigmoid(b).requires_grad_(True)
    v, dout = x["v"].double(), x["dout"].double()
    new, states, ends, outs, t = [], {}, {}, [], 0
    for L in lens:
        s = torch.zeros(hv, dk, dv, dtype=torch.float64)
        for i in range(L):
            if i % 64 == 0:
                s = s * 1.0                              # (the state between two chunks, apart from its use in the last row's output)
                if s.requires_grad:
                    s.retain_grad()
                states[t] = s
            s = s * torch.exp(g[t])[:, None, None]
            n = beta[t][:, None] * (v[t] - (s * k[t][:, :, None]).sum(1))
            n.retain_grad()
            new.append(n)
            s = s + k[t][:, :, None] * n[:, None, :]
            outs.append(scale * (s * q[t][:, :, None]).sum(1))
            t += 1
    (torch.stack(outs) * dout).sum().backward()
    N, dR, gd, bd = torch.stack(new).detach(), torch.stack([n.grad for n in new]), g.detach(), beta.detach()
    err_g = torch.zeros(T, hv, dtype=torch.float64)
    t = 0
    for L in lens:
        for c0 in range(t, t + L, 64):
            c1 = min(c0 + 64, t + L)
            rows = slice(c0, c1)
            n = c1 - c0
            heads = lambda y: y[rows].transpose(0, 1)    # (Hv, rows, ..)
            G = heads(gd).cumsum(1)
            low = torch.ones(n, n, dtype=torch.float64).tril()
            E = torch.exp(torch.where(low > 0, G[:, :, None] - G[:, None, :], 0.0)) * low
            K, Q, bt = heads(k), heads(q), heads(bd)
            kk, qk = K @ K.mT, Q @ K.mT
            Tm = torch.linalg.inv(torch.eye(n, dtype=torch.float64) + bt[..., None] * E * kk * low.tril(-1))
            Nr, dRr, dO = heads(N), heads(dR), heads(dout)
            Nabs = Tm.abs() @ torch.linalg.solve(Tm, Nr).abs()
            dRabs = Tm.mT.abs() @ torch.linalg.solve(Tm.mT, dRr).abs()
            X = scale * E * (dO.abs() @ Nabs.mT) * qk.abs()
            Z = bt[..., None] * E * (dRabs @ Nabs.mT) * kk.abs() * low.tril(-1)
            pairs = X + Z
            S0 = states[c0].detach().abs()
            dS1 = states[c1].grad.abs() if c1 < t + L else torch.zeros_like(S0)
            eg, left = torch.exp(G)[..., None], torch.exp(G[:, -1:] - G)[..., None]
            own = ((scale * eg * (Q.abs() @ S0)) * dO.abs()).sum(-1) + (bt[..., None] * eg * (K.abs() @ S0) * dRabs).sum(-1)
            last = (left * (K.abs() @ dS1) * Nabs).sum(-1)
            whole = torch.exp(G[:, -1]) * (S0 * dS1).sum((-1, -2))
            # dG_i: its pairs as a row and as a column, the states' products, and at the last row what belongs to the chunk's end
            err_i = 2.0 ** -16 * (pairs.sum(-1) + pairs.sum(-2)) + 2.0 ** -8 * (own + last)
            err_i[:, -1] += 2.0 ** -8 * (last.sum(-1) + whole)
            err_g[rows] = err_i.flip(1).cumsum(1).flip(1).transpose(0, 1)
        t += L
    dg, dbeta = g.grad, beta.grad
    slope = -rate * torch.sigmoid(z)
    da, err_a = slope * dg, slope.abs() * (err_g + 2.0 ** -18 * dg.abs())
    dlog, err_log = (gd * dg).sum(0), (gd.abs() * (err_g + 2.0 ** -18 * dg.abs())).sum(0)
    db = bd * (1 - bd) * dbeta
    err_b = GRAD * ((1 - bd) * (dR * N).abs().sum(-1)) + 2.0 ** -23 * (dR * N).abs().sum(-1)
    return {"a": (da, err_a), "b": (db, err_b), "a_log": (dlog, err_log), "dt_bias": (da.sum(0), err_a.sum(0))}


def held(got, exact):
    for n, (want, err) in exact.items():
        g = got[n].double()
        assert torch.isfinite(g).all(), n
        over = (g - want).abs() - err - 1e-30
        assert (over <= 0).all(), (n, float((g - want).abs().max()), float(err[over > 0].min()), int((over > 0).sum()))


CORNERS = {"plain": {}, "same_key": dict(k=lambda t: t[:1].expand_as(t).contiguous(), a=lambda t: t * 0 - 20, b=lambda t: t * 0 + 8),
           "no_decay": dict(a=lambda t: t * 0 - 1e30), "full_decay": dict(a=lambda t: t * 0 + 3e4), "strong_writes": dict(b=lambda t: t * 0 + 30),
           "one_reset": dict(a=lambda t: torch.where((torch.arange(t.shape[0]) % 50 == 20)[:, None], torch.full_like(t, 3e4), t)),
           "no_writes": dict(b=lambda t: t * 0 - 200)}


@pytest.mark.parametrize("kind", CORNERS)
@pytest.mark.parametrize("lens,hk,hv,dk,dv", [([200], 1, 2, 64, 64), ([0] * 250 + [90, 40] + [0] * 4, 2, 4, 72, 128), ([1] * 70, 1, 2, 64, 64)],
                         ids=["one", "many", "rows"])
def test_decay_gradients_in_the_corners(kind, lens, hk, hv, dk, dv):
    """Every row's da and db and the parameters' sums: finite, and off by no more than what the terms' roundings add up to."""
    _log(f"{kind} {len(lens)} sequences")
    x = inputs(sum(lens), hk, hv, dk, dv, seed=61, dtype=torch.float32, **CORNERS[kind])
    held(grads_of(x, lens)[1], decay_gradients(x, lens))


@pytest.mark.parametrize("lens,hv,d", [([300], 2, 128), ([90] * 12, 32, 128), ([400, 100], 2, 64)], ids=["columns", "heads", "small"])
def test_outputs_are_the_rounded_exact_ones(lens, hv, d):
    """The output and dv pass through operands of two bf16 only.  Four of them, each 2^-18 / sqrt(3) of its terms in the mean square, the terms up to four times
    their sum: 1.8e-5 of a result, which lies so close to the border between two bf16 (2^-8 to 2^-7 of it apart) once in 300 times.  An operand of one
    bf16 would turn every fifth result.  Held to ten times the first."""
    _log(f"rounded, {len(lens)} x {lens[0]}, {hv} heads of {d}")
    x = inputs(sum(lens), hv // 2, hv, d, d, seed=71)
    leaves = {n: x[n].double().requires_grad_(True) for n in NAMES}
    o, _ = R.gated_delta_rule(*leaves.values(), lens)
    dv, = torch.autograd.grad(o, leaves["v"], x["dout"].double())
    got, grads = grads_of(x, lens)
    for name, a, b in (("out", got, o), ("dv", grads["v"], dv)):
        turned = float((a != b.detach().bfloat16()).float().mean())
        assert turned <= 1 / 30, (name, turned)


def test_bits_past_two_to_the_31():
    """The last sequences of a batch whose tensors pass 2^31 elements, and of one that ends soon; their lengths split the walks alike: the same to the bit."""
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GB of free device memory")
    from tests.test_gpu_layer_offsets import rows
    hk, hv, d, T, tail = 4, 32, 128, 530_000, [2000, 1999, 2001]
    n = sum(tail)
    q, k, v, dout, a, b = rows(T, hk, d), rows(T, hk, d), rows(T, hv, d), rows(T, hv, d), rows(T, hv), rows(T, hv)
    par = torch.zeros(2, hv, device=DEV, dtype=torch.bfloat16).unbind(0)

    def run(first, take):
        leaves = [take(t).requires_grad_(True) for t in (q, k, v, a, b)]
        o = V.gated_delta_rule(*leaves, *par, cu_of([first] + tail))
        return [o.detach()[-n:].clone()] + [t[-n:].clone() for t in torch.autograd.grad(o, leaves, take(dout))]

    want = run(20_000, lambda t: t[-20_000 - n:].clone())
    for x, y in zip(run(T - n, lambda t: t), want):
        assert torch.equal(x, y)
    torch.cuda.empty_cache()
