"""The gated delta rule: value heads of one key head do not touch each other."""
import pytest
import torch

import vlm_training_amd as V
from tests.test_gpu_delta import DEV, NAMES, cu_of, inputs

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


@pytest.mark.parametrize("row", [5, 40, 100, 190])
@pytest.mark.parametrize("lens,hv,d", [([200], 2, 128), ([200] + [3] * 40, 2, 64), ([200] + [0] * 63, 16, 128)], ids=["long", "columns", "heads"])
def test_what_is_not_finite_leaves_rows_before_its_half_chunk(lens, hv, d, row):
    """A row's k, v, a or b reaches its own 32-row half of a chunk and what comes behind, its q the row alone."""
    _log(f"not finite in row {row} of {len(lens)} sequences")
    x = {n: t.to(DEV) for n, t in inputs(sum(lens), hv // 2, hv, d, d, seed=81).items()}
    run = lambda: V.gated_delta_rule(*(x[n] for n in NAMES), cu_of(lens))
    want = run()
    for n in ("k", "v", "a", "b"):
        keep = x[n][row].clone()
        x[n][row] = float("nan")
        got = run()
        x[n][row] = keep
        lo = row // 32 * 32
        assert torch.equal(got[:lo], want[:lo]) and torch.equal(got[200:], want[200:]), n
        assert not torch.isfinite(got[row]).any(), n
    x["q"][row] = float("inf")
    got = run()
    assert torch.equal(got[:row], want[:row]) and torch.equal(got[row + 1:], want[row + 1:])
