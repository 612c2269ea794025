"""The attention layers' serving form behind thousands of tokens on small pages: a prompt, a chunk whose walk's pieces begin anywhere among the pages, then single tokens, against the
packed forward of the whole sequences.

The projections' rows may be formed in another order of sums for another number of rows: q and k are then off by a step of bf16, 2^-8, each, a logit by up to 2^-7 |q||k| D^-0.5 = 2^-7 D^0.5
(normed rows: 0.09 at head_dim 128, 0.125 at 256), a weight by that and the sum's: 0.25.  A row's distance from the forward's is held to a quarter of its length, in the rows of the chunk by
themselves; keys from wrong pages, a tenth of all, put 0.4 of it there."""
import pytest
import torch

import vlm_training_amd as V
from tests.test_gpu_cache_layer import _layer, _offsets, _table, _tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("cls,hq,hkv,dim,R,page,lens,chunk", [(V.Qwen3VLTextAttention, 32, 8, 128, 128, 16, [4492, 300], [512, 40]), (V.Qwen3VLTextAttention, 16, 8, 64, 64, 16, [8152, 5962], [586, 167]),
                                                             (V.SelfAttention, 16, 2, 256, 64, 16, [6033], [509]), (V.SelfAttention, 16, 2, 256, 64, 32, [12191, 100], [525, 1])])
def test_a_chunk_behind_a_long_prompt(cls, hq, hkv, dim, R, page, lens, chunk):
    print(cls.__name__, hq, hkv, dim, page, lens, flush=True)
    hidden, steps, n = hq * dim, 3, len(lens)
    m = _layer(cls, hidden, hq, hkv, dim)                   # (the output projection is the identity)
    g = torch.Generator().manual_seed(2)
    full = [k + steps for k in lens]
    xs = [torch.randn(k, hidden, generator=g).bfloat16().to(DEV) for k in full]
    with torch.no_grad():
        want = m(torch.cat(xs)[None], *_tables(torch.cat([torch.arange(k) for k in full]), R), _offsets(full), max(full))[0].split(full)
    table, pages = _table(full, page)
    cache = V.KvCache.empty(pages, hkv, dim, page=page)
    done = [0] * n
    for new in [[k - c for k, c in zip(lens, chunk)], chunk] + [[1] * n] * steps:
        x = torch.cat([xs[i][done[i]:done[i] + k] for i, k in enumerate(new)])
        pos = torch.cat([torch.arange(done[i], done[i] + k) for i, k in enumerate(new)])
        ends = [d + k for d, k in zip(done, new)]
        got = m.extend(x, *_tables(pos, R), cache, table, _offsets(new), torch.tensor(ends, device=DEV))
        for i, part in enumerate(got.split(new)):
            ref = want[i][done[i]:ends[i]].double()
            off = (part.double() - ref).norm(dim=1) / ref.norm(dim=1)
            assert (off < 0.25).all(), (new, i, off.max().item(), int(off.argmax()))
        done = ends
