"""The gated delta rule against its definition, token by token in 64 bits (oracle/delta_ref.py).

Tolerances, of the 2-norm of the error over the result's.  A rounding to bf16 is off by at most 2^-8 of the value, 2^-8 / sqrt(3) in the mean square.
Outputs: their own rounding and those of P, N and S in front of it, four in all: 2 * 2^-8 / sqrt(3) = 4.6e-3.  Gradients: up to seven operands and the
result, 6.4e-3, half as much again for sums that partly cancel: 1e-2.  Sums over all rows of signed terms (da_log, ddt_bias) cancel further; they
are held to 1e-2 of the sum of the terms' absolute values.  States (fp32) go through two bf16 each, 2^-16 of a value per product at the most, three products deep: 5e-5."""
import pytest
import torch

import vlm_training_amd as V
from oracle import delta_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAMES = ("q", "k", "v", "a", "b", "a_log", "dt_bias")
OUT, GRAD, STATE = 4.6e-3, 1e-2, 5e-5


def _log(msg):
    print(f"[delta] {msg}", flush=True)


def inputs(T, hk, hv, dk, dv, seed=0, dtype=torch.bfloat16, **fixed):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    x = {"q": rn(T, hk, dk).bfloat16(), "k": rn(T, hk, dk).bfloat16(), "v": rn(T, hv, dv).bfloat16(), "a": rn(T, hv).to(dtype), "b": rn(T, hv).to(dtype),
         "a_log": torch.log(1 + 7 * torch.rand(hv, generator=g)).to(dtype), "dt_bias": (rn(hv) - 3).to(dtype), "dout": rn(T, hv, dv).bfloat16()}
    for n, val in fixed.items():
        x[n] = val(x[n]) if callable(val) else val
    return x


def cu_of(lens, dtype=torch.int32):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=dtype, device=DEV)


def off(got, want):
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    n = want.norm()
    return float((got - want).norm() / n) if n > 0 else float((got - want).norm())


def against(x, lens, initial=None, dfinal=None, check=NAMES, **kw):
    T = sum(lens)
    want_x = {n: x[n].double().requires_grad_(True) for n in NAMES}
    want_s = initial.double().requires_grad_(True) if initial is not None else None
    o, s = R.gated_delta_rule(*(want_x[n][:T] if n in "qkvab" else want_x[n] for n in NAMES), lens, want_s, **kw)
    loss = (o * x["dout"][:T].double()).sum() + ((s * dfinal.double()).sum() if dfinal is not None else 0.)
    loss.backward()
    got_x = {n: x[n].to(DEV).requires_grad_(True) for n in NAMES}
    got_s = initial.to(DEV).requires_grad_(True) if initial is not None else None
    go, gs = V.gated_delta_rule(*(got_x[n] for n in NAMES), cu_of(lens), initial_state=got_s, return_final_state=True, **kw)
    torch.autograd.backward([go] + ([gs] if dfinal is not None else []), [x["dout"].to(DEV)] + ([dfinal.to(DEV)] if dfinal is not None else []))
    torch.cuda.synchronize()
    assert go.dtype == torch.bfloat16 and gs.dtype == torch.float32
    assert off(go[:T], o) <= OUT, ("out", off(go[:T], o))
    assert off(gs, s) <= STATE, ("state", off(gs, s))
    assert not go[T:].any()
    for n in check:
        g, w = got_x[n].grad, want_x[n].grad
        assert g.dtype == x[n].dtype and g.shape == x[n].shape
        if n in ("a_log", "dt_bias"):
            # every row's own share: with per-row parameters the gradient is what is summed
            rows = {m: want_x[m].detach() for m in NAMES}
            rows[n] = rows[n].expand(T, -1).clone().requires_grad_(True)
            o2, s2 = R.gated_delta_rule(*(rows[m][:T] if m in "qkvab" else rows[m] for m in NAMES), lens, want_s.detach() if want_s is not None else None, **kw) \
                if n == "dt_bias" else (None, None)
            if n == "dt_bias":
                ((o2 * x["dout"][:T].double()).sum() + ((s2 * dfinal.double()).sum() if dfinal is not None else 0.)).backward()
                total = rows[n].grad.abs().sum(0)
            else:                                        # da_log = g dg, da = -exp(a_log) sigmoid(a + dt_bias) dg
                z = want_x["a"].detach()[:T] + want_x["dt_bias"].detach()
                total = (want_x["a"].grad[:T] * torch.nn.functional.softplus(z) / torch.sigmoid(z)).abs().sum(0)
            err = (g.double().cpu() - w).abs()
            assert (err <= GRAD * total + 2.0 ** -8 * w.abs() + 1e-30).all(), (n, err, total)
            continue
        assert off(g[:T], w[:T]) <= GRAD, (n, off(g[:T], w[:T]))
        if n in "qkvab":
            assert not g[T:].any(), n
    if initial is not None:
        assert off(got_s.grad, want_s.grad) <= GRAD, ("initial", off(got_s.grad, want_s.grad))


@pytest.mark.parametrize("lens,hk,hv,dk,dv", [
    ([1], 1, 1, 8, 8),
    ([2], 1, 2, 64, 64),
    ([63, 64, 65], 1, 1, 128, 128),
    ([0, 130, 0, 1, 0], 2, 4, 64, 128),
    ([300], 2, 6, 40, 72),
    ([200, 7], 1, 3, 128, 16),
    ([129], 3, 3, 72, 128),
    ([1] * 70, 1, 2, 64, 64),                             # more sequences than a wave looks at in one step
])
def test_forward_and_backward(lens, hk, hv, dk, dv):
    _log(f"lens {lens[:6]} heads {hk}/{hv} dims {dk}/{dv}")
    one = max(lens) == 1                                  # the decay of a first row reaches nothing: its gradient is zero
    x = inputs(sum(lens), hk, hv, dk, dv, seed=sum(lens))
    against(x, lens, check=tuple(n for n in NAMES if not (one and n in ("a", "a_log", "dt_bias"))))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_states_in_and_out_and_their_gradients(dtype):
    lens = [100, 0, 33]
    x = inputs(133, 2, 4, 64, 96, seed=5, dtype=dtype)
    g = torch.Generator().manual_seed(6)
    against(x, lens, torch.randn(3, 4, 64, 96, generator=g), torch.randn(3, 4, 64, 96, generator=g))


def test_scale_and_rows_taken_as_they_are():
    x = inputs(150, 1, 2, 64, 64, seed=7, q=lambda t: (0.2 * t.float()).bfloat16(), k=lambda t: (0.1 * t.float()).bfloat16())
    against(x, [150], scale=-0.7, l2_norm=False)


def test_rows_behind_the_last_sequence_give_zeros():
    x = inputs(333, 2, 4, 64, 64, seed=8)
    against(x, [70, 60])


@pytest.mark.parametrize("kind", ["same_key", "no_decay", "full_decay", "strong_writes", "one_reset"])
def test_corners_of_the_chunk_algebra(kind):
    """Equal keys fill a chunk's triangle with ones; without decay nothing is forgotten; decays that pass fp32's range leave exact zeros."""
    T, big = 200, 3e4
    change = {"same_key": dict(k=lambda t: t[:1].expand_as(t).contiguous(), a=lambda t: t * 0 - 20, b=lambda t: t * 0 + 8),
              "no_decay": dict(a=lambda t: t * 0 - 1e30), "full_decay": dict(a=lambda t: t * 0 + big), "strong_writes": dict(b=lambda t: t * 0 + 30),
              "one_reset": dict(a=lambda t: torch.where((torch.arange(T) % 50 == 20)[:, None], torch.full_like(t, big), t))}[kind]
    x = inputs(T, 1, 2, 64, 64, seed=9, **change)
    dead = {"no_decay": ("a", "a_log", "dt_bias"), "full_decay": ("a", "a_log", "dt_bias"), "same_key": ("a", "a_log", "dt_bias"), "strong_writes": ("b",),
            "one_reset": ("a_log", "dt_bias")}[kind]      # gradients that are zero, or lie below the rounding of the terms they are sums of
    against(x, [T], check=tuple(n for n in NAMES if n not in dead))


# How the state's walk is split over workgroups goes by the number of sequences and heads (empty sequences count): two blocks of columns to a workgroup, a whole head to one
MANY = [("columns", 64, 2, 64, 96), ("columns", 64, 2, 128, 128), ("head", 64, 8, 128, 128), ("head", 256, 2, 72, 104)]


@pytest.mark.parametrize("split,n,hv,dk,dv", MANY)
def test_many_sequences(split, n, hv, dk, dv):
    _log(f"{split} {n} sequences, heads of {dk}/{dv}")
    lens = [0] * n
    for i, L in zip((0, 1, 7, n // 2, n - 3, n - 1), (64, 1, 130, 65, 200, 63)):
        lens[i] = L
    g = torch.Generator().manual_seed(n + dk)
    x = inputs(sum(lens), hv // 2, hv, dk, dv, seed=n + dv)
    against(x, lens, 0.5 * torch.randn(n, hv, dk, dv, generator=g), 0.1 * torch.randn(n, hv, dk, dv, generator=g))
    x = inputs(sum(lens) + 70, hv // 2, hv, dk, dv, seed=n)
    go, gs = V.gated_delta_rule(*(x[m].to(DEV) for m in NAMES), cu_of(lens), return_final_state=True)             # nothing is kept for a backward
    o, s = R.gated_delta_rule(*(x[m].double()[:sum(lens)] if m in "qkvab" else x[m].double() for m in NAMES), lens, None)
    assert off(go[:sum(lens)], o) <= OUT and off(gs, s) <= STATE and not go[sum(lens):].any()


@pytest.mark.parametrize("split,n,hv,dk,dv", MANY[1:3])
def test_many_sequences_captured_and_on_another_stream(split, n, hv, dk, dv):
    """The same bits eagerly, replayed, on a stream of its own, and without what a backward needs."""
    _log(f"{split} {n} sequences, captured")
    lens = [70, 1, 0, 129] + [3] * (n - 4)
    x = {m: t.to(DEV) for m, t in inputs(sum(lens), hv // 2, hv, dk, dv, seed=31).items()}
    cu = cu_of(lens)
    leaves = [x[m].clone().requires_grad_(True) for m in NAMES]

    def step():
        o, s = V.gated_delta_rule(*leaves, cu, return_final_state=True)
        return [o.detach(), s.detach(), *torch.autograd.grad(o, leaves, x["dout"])]

    want = [t.clone() for t in step()]
    with torch.no_grad():
        o, s = V.gated_delta_rule(*leaves, cu, return_final_state=True)
    assert torch.equal(o, want[0]) and torch.equal(s, want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for replay in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        other = step()                                   # eager work between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {replay}"
        assert all(torch.equal(a, b) for a, b in zip(other, want))


@pytest.mark.parametrize("lens", [[2100] + [0] * 29, [89] * 24, [27] * 80, [1900] + [5] * 299], ids=["one long", "few", "many", "many and one long"])
def test_how_lengths_choose_the_split(lens):
    """Batches of 2048 rows and more, whose lengths decide on the device"""
    hv, T = 2, sum(lens)
    _log(f"{len(lens)} sequences of up to {max(lens)}")
    g = torch.Generator().manual_seed(T)
    x = inputs(T, 1, hv, 72, 72, seed=T)
    x = {m: t.to(DEV) for m, t in x.items()}
    start = 0.5 * torch.randn(len(lens), hv, 72, 72, generator=g).to(DEV)
    cu = cu_of(lens)

    def run(rows, cu, start):
        leaves = [(x[m][rows] if m in "qkvab" else x[m]).clone().requires_grad_(True) for m in NAMES] + [start.clone().requires_grad_(True)]
        o, s = V.gated_delta_rule(*leaves[:7], cu, initial_state=leaves[7], return_final_state=True)
        grads = torch.autograd.grad([o, s], leaves, [x["dout"][rows], start])
        return [o.detach(), *grads[:5]], [s.detach(), grads[7]]

    got_rows, got_states = run(slice(0, T), cu, start)
    at = 0
    for i, L in enumerate(lens):                         # each of a few alone, where there is nothing to choose (the split leaves fp32 sums of other orders: close, not equal)
        if L and i in (0, 1, 7, len(lens) - 1):
            rows, states = run(slice(at, at + L), cu_of([L]), start[i:i + 1])
            for a, b in zip(rows, got_rows):
                assert off(b[at:at + L], a.cpu()) <= 2.0 ** -7
            for a, b in zip(states, got_states):
                assert off(b[i:i + 1], a.cpu()) <= GRAD
        elif L == 0 and i < 3:
            assert torch.equal(got_states[0][i], start[i]) and torch.equal(got_states[1][i], start[i])
        at += L


@pytest.mark.parametrize("n,hv", [(3, 4), (64, 8)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_not_finite_stays_in_its_sequence(n, hv, bad):
    """Rows behind the last sequence are not read; a sequence with such rows leaves the others as they are."""
    lens = [70] + [0] * (n - 3) + [67, 130]
    T = sum(lens)
    x = {m: t.to(DEV) for m, t in inputs(T + 40, hv // 2, hv, 128, 128, seed=41).items()}
    cu = cu_of(lens)

    def run():
        leaves = [x[m].clone().requires_grad_(True) for m in NAMES]
        o = V.gated_delta_rule(*leaves, cu)
        return [o.detach(), *torch.autograd.grad(o, leaves, x["dout"])]

    want = run()
    for m in ("q", "k", "v", "a", "b", "dout"):
        x[m][T:] = bad
    got = run()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for m in ("q", "k", "v", "a", "b", "dout"):
        x[m][70:137] = bad
    for a, b in zip(run()[:6], want[:6]):
        assert torch.equal(a[:70], b[:70]) and torch.equal(a[137:], b[137:])


@pytest.mark.parametrize("kind", ["same_key", "full_decay", "one_reset"])
@pytest.mark.parametrize("split,n,hv,dk,dv", MANY[1:3])
def test_corners_in_many_sequences(split, n, hv, dk, dv, kind):
    T, big = 200, 3e4
    change = {"same_key": dict(k=lambda t: t[:1].expand_as(t).contiguous(), a=lambda t: t * 0 - 20, b=lambda t: t * 0 + 8), "full_decay": dict(a=lambda t: t * 0 + big),
              "one_reset": dict(a=lambda t: torch.where((torch.arange(T) % 50 == 20)[:, None], torch.full_like(t, big), t))}[kind]
    x = inputs(T, 1, hv, dk, dv, seed=9, **change)
    against(x, [0] * (n - 1) + [T], check=("q", "k", "v", "b"))


def test_decay_of_minus_infinity_starts_anew():
    x = inputs(140, 1, 2, 64, 64, seed=10)
    x["a"][70] = float("inf")
    args = [x[n].to(DEV).requires_grad_(True) for n in NAMES]
    whole = V.gated_delta_rule(*args, cu_of([140]))
    parts = V.gated_delta_rule(*args, cu_of([70, 70]))
    assert off(whole.double(), parts.double().cpu()) <= OUT
    whole.backward(x["dout"].to(DEV))
    assert all(torch.isfinite(t.grad).all() for t in args) and not args[3].grad[70].any()


def test_gradients_against_differences():
    """The loss's change along a random direction of all inputs at once, by central differences of the 64-bit definition, and what the gradients say."""
    lens, g = [90, 40], torch.Generator().manual_seed(11)
    x = inputs(130, 2, 4, 64, 64, seed=12, dtype=torch.float32)
    d = {n: torch.randn(x[n].shape, generator=g, dtype=torch.float64) for n in NAMES}
    loss = lambda e: (R.gated_delta_rule(*(x[n].double() + e * d[n] for n in NAMES), lens)[0] * x["dout"].double()).sum()
    want = float(loss(1e-4) - loss(-1e-4)) / 2e-4
    args = {n: x[n].to(DEV).requires_grad_(True) for n in NAMES}
    V.gated_delta_rule(*args.values(), cu_of(lens)).backward(x["dout"].to(DEV))
    terms = torch.stack([(args[n].grad.double().cpu() * d[n]).sum() for n in NAMES])
    scale = sum(float((args[n].grad.double().cpu() * d[n]).norm()) for n in NAMES)      # rounded terms add up at random
    assert abs(float(terms.sum()) - want) <= GRAD * 3 * scale, (terms, want, scale)


def test_views_strides_and_layouts():
    """Rows inside a wider tensor, expanded and oddly placed ones give what contiguous copies give, bit for bit."""
    T, hk, hv, dk, dv = 150, 2, 4, 64, 72
    x = inputs(T, hk, hv, dk, dv, seed=13)
    plain = [x[n].to(DEV) for n in NAMES]
    want = V.gated_delta_rule(*plain, cu_of([100, 50]))
    wide = torch.cat([plain[0].flatten(1), plain[1].flatten(1), plain[2].flatten(1)], 1)
    q, k, v = wide[:, :hk * dk].unflatten(1, (hk, dk)), wide[:, hk * dk:2 * hk * dk].unflatten(1, (hk, dk)), wide[:, 2 * hk * dk:].unflatten(1, (hv, dv))
    assert torch.equal(V.gated_delta_rule(q, k, v, *plain[3:], cu_of([100, 50], torch.int64)), want)
    odd = torch.empty(T * hv * dv + 1, dtype=torch.bfloat16, device=DEV)[1:].view(T, hv, dv).copy_(plain[2])        # 2 bytes past a boundary
    turned = plain[0].transpose(0, 1).contiguous().transpose(0, 1)
    ab = torch.stack([plain[3], plain[4]], -1)
    assert torch.equal(V.gated_delta_rule(turned, plain[1], odd, ab[..., 0], ab[..., 1], *plain[5:], cu_of([100, 50])), want)
    one = V.gated_delta_rule(plain[0][:, :1].expand(T, 2, dk), plain[1], *plain[2:], cu_of([100, 50]))
    assert torch.equal(one, V.gated_delta_rule(plain[0][:, :1].repeat(1, 2, 1), plain[1], *plain[2:], cu_of([100, 50])))


def test_results_are_the_same_every_time():
    x = {n: t.to(DEV) for n, t in inputs(700, 2, 6, 128, 128, seed=14).items()}
    runs = []
    for _ in range(3):
        args = [x[n].clone().requires_grad_(True) for n in NAMES]
        o = V.gated_delta_rule(*args, cu_of([500, 200]))
        runs.append([o.detach(), *torch.autograd.grad(o, args, x["dout"])])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_a_long_sequence_in_one_piece_and_in_two():
    """The state handed over in the middle: both ways agree to what the hand-over's own products are off by."""
    x = [t.to(DEV) for n, t in inputs(5000, 1, 2, 128, 128, seed=15).items() if n in NAMES]
    whole, last = V.gated_delta_rule(*x, cu_of([5000]), return_final_state=True)
    first, mid = V.gated_delta_rule(*(t[:2077] if t.shape[0] == 5000 else t for t in x), cu_of([2077]), return_final_state=True)
    rest, end = V.gated_delta_rule(*(t[2077:] if t.shape[0] == 5000 else t for t in x), cu_of([2923]), initial_state=mid, return_final_state=True)
    assert off(torch.cat([first, rest]), whole.double().cpu()) <= OUT
    assert off(end, last.double().cpu()) <= STATE


@pytest.mark.parametrize("B,hk,hv,dk,dv,dtype", [(1, 1, 1, 8, 8, torch.bfloat16), (3, 2, 4, 128, 128, torch.float32), (5, 1, 3, 40, 72, torch.bfloat16),
                                                 (2, 2, 2, 64, 104, torch.float32)])
def test_single_tokens(B, hk, hv, dk, dv, dtype):
    """Steps against the definition (fp32 throughout: the output's rounding alone, the state to a few fp32 roundings per step)."""
    _log(f"step B {B} heads {hk}/{hv} dims {dk}/{dv}")
    g = torch.Generator().manual_seed(16)
    state = torch.randn(B, hv, dk, dv, generator=g)
    pool = torch.full((2 * B, hv, dk, dv), 7.0, device=DEV)
    got = pool[1::2]                                      # requests apart from each other in a larger pool
    got.copy_(state)
    want = state.double()
    for step in range(3):
        x = inputs(B, hk, hv, dk, dv, seed=17 + step, dtype=dtype)
        o = V.gated_delta_step(*(x[n].to(DEV) for n in NAMES), got)
        wo, want = R.gated_delta_rule(*(x[n].double() for n in NAMES), [1] * B, want)
        assert off(o, wo) <= 2.0 ** -8
        assert off(got, want) <= (step + 1) * 8 * 2.0 ** -24
    assert (pool[::2] == 7.0).all()


def test_steps_go_on_where_the_packed_rows_end():
    lens, more = [37, 100], 4
    x = inputs(sum(lens) + 2 * more, 2, 4, 64, 64, seed=20)
    whole = {n: x[n].to(DEV) for n in NAMES}
    full = V.gated_delta_rule(*whole.values(), cu_of([lens[0] + more, lens[1] + more]))
    rows = torch.cat([torch.arange(lens[0]), torch.arange(lens[0] + more, sum(lens) + more)])
    head = [whole[n][rows.to(DEV)] if n in "qkvab" else whole[n] for n in NAMES]
    _, state = V.gated_delta_rule(*head, cu_of(lens), return_final_state=True)
    for i in range(more):
        at = torch.tensor([lens[0] + i, sum(lens) + more + i], device=DEV)
        o = V.gated_delta_step(*(whole[n][at] if n in "qkvab" else whole[n] for n in NAMES), state)
        assert off(o, full[at].double().cpu()) <= OUT


def test_captured_training_step_and_decoding_step():
    """Captured once, replayed with the program's own work between the replays, equal to the eager results each time."""
    x = {n: t.to(DEV) for n, t in inputs(300, 2, 4, 64, 128, seed=21).items()}
    cu = cu_of([200, 0, 100])
    leaves = [x[n].clone().requires_grad_(True) for n in NAMES]

    def step():
        o = V.gated_delta_rule(*leaves, cu)
        return [o.detach(), *torch.autograd.grad(o, leaves, x["dout"])]

    state = torch.randn(300, 4, 64, 128, device=DEV)
    start = state.clone()

    def token():
        with torch.no_grad():
            return V.gated_delta_step(*leaves, state)

    want = [t.clone() for t in step()]
    want_o = token().clone()
    want_s = state.clone()
    state.copy_(start)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        token()
    torch.cuda.current_stream().wait_stream(side)
    train, decode = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(train):
        got = step()
    with torch.cuda.graph(decode):
        got_o = token()
    for replay in range(4):
        for t in got:
            t.zero_()
        train.replay()
        state.copy_(start)
        decode.replay()
        other = step()                                   # eager work between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {replay}"
        assert all(torch.equal(a, b) for a, b in zip(other, want))
        assert torch.equal(got_o, want_o) and torch.equal(state, want_s)


def test_two_calls_at_once_on_two_streams():
    xs = [{n: t.to(DEV) for n, t in inputs(900, 2, 4, 64, 64, seed=s).items()} for s in (22, 23)]
    cu = cu_of([900])
    want = [V.gated_delta_rule(*(x[n] for n in NAMES), cu) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for x, st in zip(xs, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append([V.gated_delta_rule(*(x[n] for n in NAMES), cu) for _ in range(3)])
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, o) for o in g)


def test_empty_batches():
    x = [t.to(DEV).requires_grad_(True) for n, t in inputs(0, 2, 4, 64, 64).items() if n in NAMES]
    first = torch.randn(2, 4, 64, 64, device=DEV)
    o, s = V.gated_delta_rule(*x, cu_of([0, 0]), initial_state=first, return_final_state=True)
    assert o.shape == (0, 4, 64, 64)[:1] + (4, 64) and torch.equal(s, first)
    o.sum().backward()
    assert not x[5].grad.any() and not x[6].grad.any()
    with torch.no_grad():
        assert V.gated_delta_step(*x, torch.empty(0, 4, 64, 64, device=DEV)).shape == (0, 4, 64)


def test_only_some_inputs_need_a_gradient():
    x = {n: t.to(DEV) for n, t in inputs(100, 1, 2, 64, 64, seed=24).items()}
    every = [x[n].clone().requires_grad_(True) for n in NAMES]
    want = torch.autograd.grad(V.gated_delta_rule(*every, cu_of([100])), every, x["dout"])
    some = [x[n].clone().requires_grad_(n in ("v", "dt_bias")) for n in NAMES]
    V.gated_delta_rule(*some, cu_of([100])).backward(x["dout"])
    assert torch.equal(some[2].grad, want[2]) and torch.equal(some[6].grad, want[6]) and some[0].grad is None


def test_refusals():
    x = [t.to(DEV) for n, t in inputs(64, 2, 4, 64, 64, seed=25).items() if n in NAMES]
    cu, state = cu_of([64]), torch.zeros(64, 4, 64, 64, device=DEV)

    def swap(i, t):
        return x[:i] + [t] + x[i + 1:]

    for bad in (swap(0, x[0].float()), swap(1, x[1][:32]), swap(2, x[2][:, :3]), swap(3, x[3][:, :2]), swap(4, x[4].half()), swap(5, x[5][:2]), swap(2, x[2][0])):
        with pytest.raises(ValueError):
            V.gated_delta_rule(*bad, cu)
        with pytest.raises(ValueError):
            V.gated_delta_step(*bad, state)
    with pytest.raises(ValueError):
        V.gated_delta_rule(*x, cu, scale=0.0)
    with pytest.raises(ValueError):
        V.gated_delta_rule(*x, cu[:1])
    with pytest.raises(ValueError):
        V.gated_delta_rule(*x, cu, initial_state=torch.zeros(2, 4, 64, 64, device=DEV))
    with pytest.raises(ValueError):
        V.gated_delta_rule(*x, cu, initial_state=torch.zeros(1, 4, 64, 64, device=DEV, dtype=torch.bfloat16))
    wide = torch.zeros(64, 2, 136, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="multiples of 8 up to 128"):
        V.gated_delta_rule(wide, wide, *x[2:], cu)
    with pytest.raises(RuntimeError, match="multiples of 8 up to 128"):
        V.gated_delta_rule(wide[..., :12], wide[..., :12], *x[2:], cu)
    with pytest.raises(RuntimeError, match="GPU only"):
        V.gated_delta_rule(*(t.cpu() for t in x), cu.cpu())
    with pytest.raises(ValueError, match="in place"):
        V.gated_delta_step(*x, state.transpose(2, 3))
    with pytest.raises(ValueError, match="in place"):
        V.gated_delta_step(*x, state[:1].expand(64, 4, 64, 64))
    with pytest.raises(ValueError, match="backward"):
        V.gated_delta_step(x[0].clone().requires_grad_(True), *x[1:], state)
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises(NotImplementedError):
        V.gated_delta_rule(fwAD.make_dual(x[0].float(), x[0].float()), *x[1:], cu)
