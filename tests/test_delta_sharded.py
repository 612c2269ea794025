"""A linear-attention layer under tensor parallelism: in_proj_qkv's rows are [q | k | v], so that a column shard of them is not whole heads of each.  Runs
without a GPU: what cannot be right is refused before any kernel."""
import os
from types import SimpleNamespace

import pytest
import torch

from vlm_training_amd.layers import DeltaState, GatedDeltaNet

CFG = SimpleNamespace(hidden_size=64, linear_num_key_heads=2, linear_num_value_heads=8, linear_key_head_dim=16, linear_value_head_dim=16, linear_conv_kernel_dim=4,
                      rms_norm_eps=1e-6)


def shard_worker(rank, port, out):
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import Replicate, Shard, distribute_tensor
    from torch.distributed.tensor.parallel import ColwiseParallel, parallelize_module
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2)
    try:
        mesh = init_device_mesh("cpu", (2,))
        cu, x = torch.tensor([0, 5], dtype=torch.int32), torch.zeros(1, 5, 64)
        state = DeltaState(torch.zeros(5, 192, 3, dtype=torch.bfloat16), torch.zeros(5, 8, 16, 16))
        seen = []

        def texts(layer):
            for call in (lambda: layer(x, cu), lambda: layer.step(x[0], state)):
                try:
                    call()
                    seen.append("ran")
                except Exception as e:
                    seen.append(f"{type(e).__name__}: {e}")

        for local in (True, False):
            layer = GatedDeltaNet(CFG)
            parallelize_module(layer, mesh, {n: ColwiseParallel(use_local_output=local) for n in ("in_proj_qkv", "in_proj_z", "in_proj_a", "in_proj_b")})
            texts(layer)
        layer = GatedDeltaNet(CFG)                       # the convolution's channels alone
        layer.conv1d.weight = torch.nn.Parameter(distribute_tensor(layer.conv1d.weight.detach(), mesh, [Shard(0)]))
        texts(layer)
        layer = GatedDeltaNet(CFG)                       # the same on every rank: nothing is split (and there is no GPU here)
        layer.conv1d.weight = torch.nn.Parameter(distribute_tensor(layer.conv1d.weight.detach(), mesh, [Replicate()]))
        texts(layer)
        out.put((rank, seen))
    finally:
        dist.destroy_process_group()


def test_column_shards_of_the_packed_projection_are_refused():
    import torch.multiprocessing as mp
    ctx = mp.get_context("spawn")
    out = ctx.Queue()
    port = 29650 + os.getpid() % 200
    workers = [ctx.Process(target=shard_worker, args=(r, port, out)) for r in range(2)]
    for w in workers:
        w.start()
    results = [out.get(timeout=240) for _ in workers]
    for w in workers:
        w.join(60)
        assert w.exitcode == 0
    for _, seen in results:
        assert len(seen) == 8
        for text in seen[:6]:
            assert text.startswith("ValueError") and "whole heads" in text, seen
        for text in seen[6:]:
            assert "GPU only" in text, seen


def test_heads_that_do_not_fit_each_other_are_refused():
    """in_proj_z of half the value heads beside an in_proj_qkv of all: the widths alone would pass as other heads."""
    layer, half = GatedDeltaNet(CFG), GatedDeltaNet(SimpleNamespace(**{**vars(CFG), "linear_num_value_heads": 4, "linear_num_key_heads": 1}))
    for n in ("in_proj_z", "in_proj_a", "in_proj_b", "A_log", "dt_bias"):
        setattr(layer, n, getattr(half, n))
    with pytest.raises(ValueError, match="heads"):
        layer(torch.zeros(1, 5, 64), torch.tensor([0, 5], dtype=torch.int32))
    whole = GatedDeltaNet(CFG)                           # a head-sharded layer whose rows were sorted by head passes
    for n in ("in_proj_qkv", "in_proj_z", "in_proj_a", "in_proj_b", "conv1d", "A_log", "dt_bias"):
        setattr(whole, n, getattr(half, n))
    with pytest.raises(RuntimeError, match="GPU only"):
        whole(torch.zeros(1, 5, 64), torch.tensor([0, 5], dtype=torch.int32))


def test_every_placement_that_splits_rows_counts():
    """Strided shards, as they come of two kinds of parallelism at once, are not of the plain ones' class."""
    from torch.distributed.tensor import Partial, Replicate, Shard
    from torch.distributed.tensor.placement_types import _StridedShard
    from vlm_training_amd import dtensor_utils

    class Weight:                                        # (what is looked at of a DTensor)
        def __init__(self, *placements):
            self.placements, self.device_mesh = placements, SimpleNamespace(size=lambda i: 1 if i == 2 else 4)

    seen, dtensor_utils.DTensor = dtensor_utils.DTensor, Weight
    try:
        split = lambda *p: dtensor_utils._column_sharded(Weight(*p))
        assert split(Shard(0)) and split(_StridedShard(0, split_factor=2)) and split(Replicate(), Shard(0)) and split(Shard(1), _StridedShard(0, split_factor=4))
        assert not split(Replicate()) and not split(Shard(1)) and not split(Partial()) and not split(Replicate(), Shard(1), Shard(0)) and not split()
    finally:
        dtensor_utils.DTensor = seen
    assert not dtensor_utils._column_sharded(torch.zeros(4, 4)) and not dtensor_utils._column_sharded(None)
