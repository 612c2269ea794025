"""A linear-attention layer with DTensor projections, and one with the rows of some of the heads: what each rank of a head-sharded layer runs."""
import copy

import pytest
import torch

from tests.test_gpu_delta_layer import CFG, DEV, build
from tests.test_gpu_layers import _one_rank_cuda_mesh

pytestmark = pytest.mark.gpu


def test_dtensor_projections_on_one_rank_give_the_plain_layer():
    """Column-parallel projections with DTensor outputs and a row-parallel out_proj on a mesh of one rank: the local shard is the whole tensor, so outputs and
    gradients equal the plain layer's bit for bit."""
    import torch.distributed as dist
    from torch.distributed.tensor import DTensor
    from torch.distributed.tensor.parallel import ColwiseParallel, RowwiseParallel, parallelize_module
    plain = build()[0].to(DEV)
    x = torch.randn(1, 90, 256, device=DEV).bfloat16()
    cu = torch.tensor([0, 50, 90], dtype=torch.int32, device=DEV)
    dy = torch.randn(1, 90, 256, device=DEV).bfloat16()
    mesh, created = _one_rank_cuda_mesh()
    try:
        tp = copy.deepcopy(plain)
        parallelize_module(tp, mesh, {**{n: ColwiseParallel(use_local_output=False) for n in ("in_proj_qkv", "in_proj_z", "in_proj_a", "in_proj_b")},
                                      "out_proj": RowwiseParallel()}, src_data_rank=None)      # (shards are taken from the local copy: nothing is scattered)
        assert isinstance(tp.in_proj_qkv.weight, DTensor)
        a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
        want, got = plain(a, cu), tp(b, cu)
        got = got.to_local() if isinstance(got, DTensor) else got
        want.backward(dy)
        got.backward(dy)
        assert torch.equal(got, want) and torch.equal(a.grad, b.grad)
        for (n, p), q in zip(plain.named_parameters(), tp.parameters()):
            g = q.grad.to_local() if isinstance(q.grad, DTensor) else q.grad
            assert torch.equal(g, p.grad), n
    finally:
        if created:
            dist.destroy_process_group()


def test_layers_of_half_the_heads_each_add_up_to_the_whole():
    """Two layers with the rows of one key head and its value heads each: their outputs add up to the whole layer's, up to the three roundings to bf16 (2^-8 of the
    values each, out_proj's two halves and the whole)."""
    whole = build()[0].to(DEV)
    hk, hv, d = CFG.linear_num_key_heads, CFG.linear_num_value_heads, CFG.linear_key_head_dim
    x = torch.randn(1, 90, 256, device=DEV).bfloat16()
    cu = torch.tensor([0, 50, 90], dtype=torch.int32, device=DEV)
    with torch.no_grad():
        total = 0
        for r in range(2):
            half = copy.deepcopy(whole)
            keys = torch.arange(hk * d, device=DEV).chunk(2)[r]
            values, heads = torch.arange(hv * d, device=DEV).chunk(2)[r], torch.arange(hv, device=DEV).chunk(2)[r]
            mixed = torch.cat([keys, hk * d + keys, 2 * hk * d + values])
            for name, rows in (("in_proj_qkv", mixed), ("in_proj_z", values), ("in_proj_a", heads), ("in_proj_b", heads), ("conv1d", mixed)):
                lin = getattr(half, name)
                lin.weight = torch.nn.Parameter(lin.weight[rows])
            half.A_log, half.dt_bias = torch.nn.Parameter(half.A_log[heads]), torch.nn.Parameter(half.dt_bias[heads])
            half.out_proj.weight = torch.nn.Parameter(half.out_proj.weight[:, values])
            total = total + half(x, cu).float()
        want = whole(x, cu).float()
    assert float((total - want).norm()) <= 3 * 2.0 ** -8 * float(want.norm())
