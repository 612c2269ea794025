"""How exactly the chunk gradients take what the walks leave them."""
import pytest
import torch

import vlm_training_amd as V
from oracle import delta_ref as R
from tests.test_gpu_delta import DEV, NAMES, cu_of, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,hv,dk,dv", [(64, 2, 128, 128), (37, 4, 64, 128), (64, 3, 40, 72)])
def test_gradients_of_one_chunk_between_states_of_few_bits(rows, hv, dk, dv):
    """One chunk whose states at both ends are bf16 numbers: all other operands are two bf16, each off by 2^-18, so dq and dk are the exact ones rounded but for results
    that lie within some 2^-15 of themselves of the border between two bf16 (2^-8 to 2^-7 apart): one in 100.  An operand of one bf16 would turn every fifth;
    held to one in 25.  da and db are fp32 sums of the same products, 2^-18 of terms up to 64 times the result: 2^-12."""
    g = torch.Generator().manual_seed(rows + dk)
    few = lambda *s: torch.randn(*s, generator=g).bfloat16().float()
    x = inputs(rows, 1, hv, dk, dv, seed=3, dtype=torch.float32)
    first, dlast = 0.5 * few(1, hv, dk, dv), 0.5 * few(1, hv, dk, dv)
    want = {n: x[n].double().requires_grad_(True) for n in NAMES}
    o, s = R.gated_delta_rule(*want.values(), [rows], first.double())
    ((o * x["dout"].double()).sum() + (s * dlast.double()).sum()).backward()
    got = {n: x[n].to(DEV).requires_grad_(True) for n in NAMES}
    o, s = V.gated_delta_rule(*got.values(), cu_of([rows]), initial_state=first.to(DEV), return_final_state=True)
    torch.autograd.backward([o, s], [x["dout"].to(DEV), dlast.to(DEV)])
    for n in ("q", "k", "v"):
        turned = float((got[n].grad.cpu() != want[n].grad.bfloat16()).float().mean())
        assert turned <= 1 / 25, (n, turned)
    for n in ("a", "b"):
        w = want[n].grad
        assert float((got[n].grad.double().cpu() - w).norm()) <= 2.0 ** -12 * float(w.norm()), n
