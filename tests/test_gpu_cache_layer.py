"""The attention layers' serving form: prompts in chunks and single tokens through the paged cache against the packed forward of the whole sequences.

Tolerance where the output projection is the identity: q and k are the same bits on both sides, and each side's attention is off by half a step of bf16 (2^-8) of its value and, through
the rounding of its probabilities, of the weighted mean of |v|, which the largest |v| bounds; a gate in (0, 1) rounds once more: 2 * (2^-8 (2 |y| + |v|)) between the two."""
from types import SimpleNamespace

import pytest
import torch

import vlm_training_amd as V
from tests.util import cosine

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _offsets(parts):
    return torch.tensor([sum(parts[:i]) for i in range(len(parts) + 1)], dtype=torch.int32, device=DEV)


def _tables(positions, R):
    ang = torch.outer(positions.float(), 1.0 / (1e4 ** (torch.arange(0, R, 2, dtype=torch.float32) / R)))
    emb = torch.cat((ang, ang), -1).to(DEV)
    return emb.cos().bfloat16(), emb.sin().bfloat16()


def _layer(cls, hidden, hq, hkv, dim, seed=0, identity=True):
    torch.manual_seed(seed)
    m = cls(SimpleNamespace(hidden_size=hidden, num_attention_heads=hq, num_key_value_heads=hkv, head_dim=dim, rms_norm_eps=1e-6)).to(DEV).bfloat16()
    if identity:
        with torch.no_grad():
            m.o_proj.weight.copy_(torch.eye(hidden))
    return m


def _table(lens, page, seed=0):
    need = [(n + page - 1) // page for n in lens]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed)).int()
    table, at = torch.full((len(lens), max(need)), -1, dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table.to(DEV), sum(need)


def _schedule(lens):
    """New tokens of each request, call by call: chunks of prompts beside single tokens, requests that wait."""
    left, calls, k = list(lens), [], 0
    while any(left):
        new = [min(n, (37, 1, 0, 5, 90)[(i + k) % 5]) for i, n in enumerate(left)]
        left = [n - m for n, m in zip(left, new)]
        calls.append(new)
        k += 1
    return calls


def _run(call, xs, lens, R):
    """``call(x, cos, sin, cu, lengths, new)`` over the schedule; the outputs of each request in order."""
    done, outs = [0] * len(lens), [[] for _ in lens]
    for new in _schedule(lens):
        if not any(new):
            continue
        x = torch.cat([xs[i][done[i]:done[i] + m] for i, m in enumerate(new)])
        pos = torch.cat([torch.arange(done[i], done[i] + m) for i, m in enumerate(new)])
        done = [d + m for d, m in zip(done, new)]
        y = call(x, *_tables(pos, R), _offsets(new), torch.tensor(done, dtype=torch.int32, device=DEV), new)
        for o, part in zip(outs, y.split(new)):
            o.append(part)
    return torch.cat([torch.cat(o) for o in outs])


@pytest.mark.parametrize("cls,hq,hkv,dim,R,page", [(V.Qwen3VLTextAttention, 8, 2, 64, 64, 16), (V.Qwen3VLTextAttention, 4, 4, 128, 128, 64), (V.SelfAttention, 4, 1, 256, 64, 32)])
def test_chunks_and_steps_give_what_the_whole_sequences_give(cls, hq, hkv, dim, R, page):
    print(cls.__name__, hq, hkv, dim, page, flush=True)
    lens, hidden = [200, 7, 64, 131], hq * dim
    m = _layer(cls, hidden, hq, hkv, dim)
    g = torch.Generator().manual_seed(1)
    xs = [torch.randn(n, hidden, generator=g).bfloat16().to(DEV) for n in lens]
    pos = torch.cat([torch.arange(n) for n in lens])
    with torch.no_grad():
        want = m(torch.cat(xs)[None], *_tables(pos, R), _offsets(lens), max(lens))[0]
        most_v = m.v_proj(torch.cat(xs)).abs().max().item()
    table, pages = _table(lens, page)
    cache = V.KvCache.empty(pages, hkv, dim, page=page)
    got = _run(lambda x, cos, sin, cu, lengths, new: m.extend(x, cos, sin, cache, table, cu, lengths, max_new=max(new), max_length=max(lens)), xs, lens, R)
    err, bound = (got.double() - want.double()).abs(), 2.0 ** -7 * (2 * want.double().abs() + most_v)
    assert (err <= bound).all(), (err - bound).max()
    # without bounds, (1, T, hidden), a second time over the same pages (which are written with the same rows again)
    again = _run(lambda x, cos, sin, cu, lengths, new: m.extend(x[None], cos[None], sin[None], cache, table, cu.long(), lengths)[0], xs, lens, R)
    assert ((again.double() - want.double()).abs() <= bound).all()
    # what the cache holds: the values as the projection gave them
    _, v = V.kv_cache_read(cache, table, _offsets(lens), sum(lens))
    with torch.no_grad():
        assert torch.equal(v, torch.cat([m.v_proj(x) for x in xs]).unflatten(-1, (-1, dim))) or (v.float() - m.v_proj(torch.cat(xs)).unflatten(-1, (-1, dim)).float()).abs().max() < 2.0 ** -6 * most_v


def test_a_hybrid_stack_answers():
    """A linear-attention layer and a full-attention one with an 8-bit cache, with residuals: prompts, then token by token, against the packed forward.  e4m3 keys and values are off by 2^-4 at
    most, 2^-5 in the mean square: an eighth of that is left after a softmax over hundreds of keys; held to a cosine of 0.998 (an error of 6 %)."""
    hidden, lens, steps, page = 256, [150, 33, 80], 12, 32
    full = [n + steps for n in lens]
    attn = _layer(V.SelfAttention, hidden, 4, 2, 64, seed=3, identity=False)
    torch.manual_seed(4)
    delta = V.GatedDeltaNet(SimpleNamespace(hidden_size=hidden, linear_num_key_heads=2, linear_num_value_heads=4, linear_key_head_dim=64, linear_value_head_dim=64,
                                            linear_conv_kernel_dim=4, rms_norm_eps=1e-6)).to(DEV).bfloat16()
    g = torch.Generator().manual_seed(5)
    xs = [torch.randn(n, hidden, generator=g).bfloat16().to(DEV) for n in full]
    with torch.no_grad():
        x = torch.cat(xs)[None]
        h = x + delta(x, _offsets(full))
        want = (h + attn(h, *_tables(torch.cat([torch.arange(n) for n in full]), 64), _offsets(full), max(full)))[0]
    table, pages = _table(full, page)
    cache = V.KvCache.empty(pages, 2, 64, page=page, dtype=torch.float8_e4m3fn)
    with torch.no_grad():
        x = torch.cat([a[:n] for a, n in zip(xs, lens)])[None]
        y, state = delta(x, _offsets(lens), return_state=True)
        h = x + y
        got = [list((h + attn.extend(h, *_tables(torch.cat([torch.arange(n) for n in lens]), 64), cache, table, _offsets(lens), torch.tensor(lens, device=DEV)))[0].split(lens))]
        for k in range(steps):
            x = torch.stack([a[n + k] for a, n in zip(xs, lens)])
            h = x + delta.step(x, state)
            pos = torch.tensor([n + k for n in lens])
            y = h + attn.extend(h, *_tables(pos, 64), cache, table, _offsets([1] * 3), (pos + 1).int().to(DEV), max_new=1, max_length=max(full))
            got.append(list(y.split([1] * 3)))
    got = torch.cat([torch.cat([call[i] for call in got]) for i in range(3)])
    for a, b in ((got, want), (got - torch.cat(xs), want - torch.cat(xs))):
        assert cosine(a.float().cpu(), b.float().cpu()) > 0.998


def test_refusals():
    m = _layer(V.SelfAttention, 128, 2, 1, 64)
    m.indexer = V.DsaIndexer(128, V.DsaConfig(4, 64, 8)).to(DEV).bfloat16()
    x = torch.zeros(1, 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(NotImplementedError):
        m.extend(x, *_tables(torch.zeros(1), 64), V.KvCache.empty(1, 1, 64), torch.zeros(1, 1, dtype=torch.int32, device=DEV), _offsets([1]), torch.ones(1, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        _layer(V.SelfAttention, 128, 2, 1, 64).extend(x, *_tables(torch.zeros(1), 64), V.KvCache.empty(1, 2, 64), torch.zeros(1, 1, dtype=torch.int32, device=DEV), _offsets([1]),
                                                      torch.ones(1, dtype=torch.int32, device=DEV))
