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
