"""The operators of a paged key/value cache: their calls, and the same in elementary torch operations.

``op`` names the operator:

* ``attend``  ``paged_attn``: the new tokens of each request (one, a few drafted ones, a chunk of a prompt) over everything the cache holds of it
* ``write``   ``kv_cache_write``: the keys and values of new tokens into the pages, a bf16 cache (the pages are what comes back)
* ``store``   the same into a cache of 8-bit values, and ``kv_cache_read`` of the rows just written: what later tokens will see of them
* ``read``    ``kv_cache_read``: the rows of a range of positions, packed, as bf16

``new`` holds the new tokens of each request (of ``read``: the rows read), ``lens`` its length with them, both comma-separated.  A cache is
(pages, kv heads, page, head_dim) for keys and for values, bf16, or e4m3 with a power of two for each row of each head; pages lie in any order.
"""
import math

import torch

own = False
DEV = "cuda"
SMALLEST = -100          # exponent of the smallest scale of a row


# ---- cases ----------------------------------------------------------------------------------------------------------
def _text(numbers):
    return ",".join(str(n) for n in numbers)


def _spread(n, lo, hi):
    """n lengths from lo to hi, even on a logarithmic scale, in an order that mixes short and long ones."""
    at = [int(round(lo * (hi / lo) ** (i / max(n - 1, 1)))) for i in range(n)]
    return [at[(i * 29) % n] for i in range(n)] if n % 29 else at


def _case(op, new, lens, hq=32, hkv=8, dim=128, page=64, kind="bf16"):
    return dict(op=op, new=_text(new), lens=_text(lens), hq=hq, hkv=hkv, dim=dim, page=page, kind=kind)


def listed():
    return [
        # one request's next token, a short conversation: all latency
        dict(_case("attend", [1], [1000]), name="attend_step_1"),
        # a serving batch's next tokens, conversations of 64 to 8192 tokens side by side
        dict(_case("attend", [1] * 64, _spread(64, 64, 8192)), name="attend_step_64"),
        # a large serving batch over an 8-bit cache: the cache passes through memory once
        dict(_case("attend", [1] * 256, _spread(256, 2048, 8192), kind="e4m3"), name="attend_step_256_8bit"),
        # one very long document and a short request beside it: a single walk of 131 072 keys if it is not split
        dict(_case("attend", [1, 1], [131072, 77], hq=16, hkv=2, dim=256, page=128), name="attend_step_131k"),
        # four drafted tokens of each request looked over at once
        dict(_case("attend", [4] * 24, _spread(24, 300, 5000), kind="e4m3"), name="attend_draft_24"),
        # a chunk of a long prompt: 2048 new tokens behind 14 336 cached ones
        dict(_case("attend", [2048], [16384]), name="attend_chunk_2k"),
        # what a scheduler with chunked prompts sends: a chunk, a short new prompt and forty requests' next tokens, 8-bit cache
        dict(_case("attend", [512, 333] + [1] * 40, [8192, 333] + _spread(40, 200, 4000), kind="e4m3"), name="attend_mixed_8bit"),
        # odd heads, head_dim, lengths and small pages; a request without new tokens, one without anything, one whose first new row has no key
        dict(_case("attend", [1, 70, 0, 3, 129, 0, 17], [1, 233, 64, 3, 1000, 0, 16], hq=6, hkv=3, dim=72, page=16), name="attend_odd"),
        # the keys and values of a prompt chunk into a bf16 cache
        dict(_case("write", [8192, 1, 4095, 100], [8192, 500, 10000, 100]), name="write_12k"),
        # the same into an 8-bit cache and back: a chunk, and one token of each request
        dict(_case("store", [8192, 1, 4095, 100], [8192, 500, 10000, 100], kind="e4m3"), name="store_12k_8bit"),
        dict(_case("store", [1] * 256, _spread(256, 100, 4000), kind="e4m3"), name="store_step_256_8bit"),
        # eight requests' cached rows packed for the operators that take packed rows, from an 8-bit cache
        dict(_case("read", [9000, 1, 700, 12000, 63, 4096, 333, 6575], [9000, 1, 1700, 12000, 64, 5000, 333, 6575], kind="e4m3"), name="read_32k_8bit"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv, dim = rng.choice([(32, 8, 128), (32, 8, 128), (16, 8, 128), (16, 2, 256), (8, 8, 64), (6, 3, 96), (16, 1, 128), (5, 1, 80)])
    page, kind = rng.choice([16, 32, 64, 64, 128, 256]), rng.choice(["bf16", "e4m3"])
    row = 2 * hkv * dim * 2
    op = rng.choice(["attend"] * 6 + ["write", "store", "read"])
    if op == "attend":
        shape = rng.choice(["step", "step", "draft", "chunk", "mixed"])
        if shape == "chunk":
            new = _log(rng, 17, 2048)
            return _case(op, [new], [new + rng.choice([0, _log(rng, 1, 14000)])], hq, hkv, dim, page, kind)
        n = _log(rng, 1, 200)
        lens = [_log(rng, 1, min(100000, 1500000000 // (row * n))) for _ in range(n)]
        if shape == "step":
            return _case(op, [1] * n, lens, hq, hkv, dim, page, kind)
        if shape == "draft":
            return _case(op, [1] + [min(rng.randint(0, 8), k) for k in lens[1:]], lens, hq, hkv, dim, page, kind)
        lens[0] = min(lens[0], 30000)
        return _case(op, [min(_log(rng, 17, 700), lens[0])] + [1] * (n - 1), lens, hq, hkv, dim, page, kind)
    n = _log(rng, 1, 300)
    new = [rng.choice([1, 1, _log(rng, 1, max(1, 15000 // n))]) for _ in range(n)]
    lens = [k + rng.choice([0, _log(rng, 1, 1000)]) for k in new]
    return _case(op, new, lens, hq, hkv, dim, page, "bf16" if op == "write" else "e4m3" if op == "store" else kind)


def _ints(text):
    return [int(n) for n in text.split(",")]


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _encode(x):
    """Rows of 32-bit values -> e4m3 values and a power of two for each row, the smallest one under which its largest value is at most 448."""
    mantissa, exponent = torch.frexp(x.abs().amax(-1))
    exponent = (exponent - torch.where(mantissa <= 0.875, 9, 8)).clamp(min=SMALLEST)
    codes = torch.ldexp(x, -exponent[..., None]).to(torch.float8_e4m3fn)
    return codes, (exponent + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _decode(codes, scale):
    if scale is None:
        return codes.float()
    return torch.ldexp(codes.float(), scale.view(torch.uint8).int()[..., None] - 127)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    new, lens = _ints(case["new"]), _ints(case["lens"])
    hq, hkv, dim, page = (case[x] for x in ("hq", "hkv", "dim", "page"))
    need = [(n + page - 1) // page for n in lens]
    pages, rows = sum(need) + 3, sum(new)
    order = torch.randperm(pages, generator=g, device=DEV).int()
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n

    def offsets(parts):
        return torch.tensor([sum(parts[:i]) for i in range(len(parts) + 1)], dtype=torch.int32, device=DEV)

    s = {"case": dict(case), "new": new, "lens": lens, "rows": rows, "table": table, "cu": offsets(new), "lengths": torch.tensor(lens, dtype=torch.int32, device=DEV),
         "first": torch.tensor([n - m for n, m in zip(lens, new)], dtype=torch.int32, device=DEV)}
    # keys are normed and rotated, one or two channels of each head larger than the rest
    loud = 1 + 2 * (torch.rand(hkv, 1, dim, generator=g, device=DEV) > 0.98)

    def pool(std):
        x = [torch.randn(min(256, pages - p), hkv, page, dim, generator=g, device=DEV) * std for p in range(0, pages, 256)]
        if case["kind"] == "bf16":
            return torch.cat([t.bfloat16() for t in x]), None
        codes, scale = zip(*(_encode(t.bfloat16().float()) for t in x))
        return torch.cat(codes), torch.cat(scale)

    s["k_pages"], s["k_scale"] = pool(loud)
    s["v_pages"], s["v_scale"] = pool(0.7)
    if case["op"] == "attend":
        s["q"] = (torch.randn(rows, hq, dim, generator=g, device=DEV) * 1.3).bfloat16()
    elif case["op"] != "read":
        # the keys come from the norm and rotation; the values lie in the projection's output
        s["k"] = (torch.randn(rows, hkv, dim, generator=g, device=DEV) * loud.transpose(0, 1)).bfloat16()
        s["v"] = (torch.randn(rows, 2 * hkv, dim, generator=g, device=DEV) * 0.7).bfloat16()[:, hkv:]
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        import vlm_training_amd as V
        cache = V.KvCache(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
        if op == "attend":
            return V.paged_attn(s["q"], cache, s["table"], s["cu"], s["lengths"], max_new=max(s["new"]), max_length=max(s["lens"]))
        if op in ("write", "store"):
            V.kv_cache_write(cache, s["k"], s["v"], s["table"], s["cu"], s["lengths"])
        if op == "write":
            return s["k_pages"], s["v_pages"]
        return V.kv_cache_read(cache, s["table"], s["cu"], s["rows"], first=s["first"])
    if op == "attend":
        return _plain_attn(s)
    if op in ("write", "store"):
        _plain_write(s)
    if op == "write":
        return s["k_pages"], s["v_pages"]
    return _plain_read(s)


# ---- the plain forms: 32 bits throughout, rounded at the end ---------------------------------------------------------
def _plain_slots(s):
    """Page and place in the page of every row."""
    seq = torch.repeat_interleave(torch.arange(len(s["new"]), device=DEV), (s["cu"][1:] - s["cu"][:-1]).long(), output_size=s["rows"])
    position = s["first"].long()[seq] + torch.arange(s["rows"], device=DEV) - s["cu"].long()[seq]
    return s["table"].long()[seq, position // s["case"]["page"]], position % s["case"]["page"]


def _plain_write(s):
    page, place = _plain_slots(s)
    for name in ("k", "v"):
        if s["case"]["kind"] == "bf16":
            s[name + "_pages"][page, :, place] = s[name]
        else:
            codes, scale = _encode(s[name].float())
            s[name + "_pages"].view(torch.uint8)[page, :, place] = codes.view(torch.uint8)
            s[name + "_scale"].view(torch.uint8)[page, :, place] = scale.view(torch.uint8)


def _plain_read(s):
    page, place = _plain_slots(s)
    out = []
    for name in ("k", "v"):
        pages, scale = s[name + "_pages"], s[name + "_scale"]
        if scale is None:
            out.append(pages[page, :, place])
        else:
            out.append(_decode(pages.view(torch.uint8)[page, :, place].view(torch.float8_e4m3fn), scale.view(torch.uint8)[page, :, place].view(torch.float8_e8m0fnu)).bfloat16())
    return tuple(out)


def _plain_attn(s):
    case, q, out, at = s["case"], s["q"], torch.empty_like(s["q"]), 0
    hq, hkv, dim, page = (case[x] for x in ("hq", "hkv", "dim", "page"))
    group = hq // hkv
    for i, (new, length) in enumerate(zip(s["new"], s["lens"])):
        if new == 0:
            continue
        mine = s["table"][i, :(length + page - 1) // page].long()

        def rows(name):
            pages, scale = s[name + "_pages"], s[name + "_scale"]
            if scale is None:
                x = pages[mine].float()
            else:
                x = _decode(pages.view(torch.uint8)[mine].view(torch.float8_e4m3fn), scale.view(torch.uint8)[mine].view(torch.float8_e8m0fnu))
            return x.transpose(0, 1).reshape(hkv, -1, dim)[:, :length]

        k, v = rows("k").transpose(1, 2).contiguous(), rows("v").contiguous()
        for lo in range(0, new, 512):
            hi = min(lo + 512, new)
            x = q[at + lo:at + hi].float().view(hi - lo, hkv, group, dim).permute(1, 0, 2, 3).reshape(hkv, -1, dim)
            logits = (x @ k) * dim ** -0.5
            limit = torch.arange(length - new + lo, length - new + hi, device=DEV).repeat_interleave(group)
            logits.masked_fill_(torch.arange(length, device=DEV) > limit[:, None], -math.inf)
            weight = torch.exp(logits - logits.amax(-1, keepdim=True))
            o = torch.where(limit[:, None] >= 0, (weight @ v) / weight.sum(-1, keepdim=True), 0.0)          # (zeros for a row without a key)
            out[at + lo:at + hi] = o.view(hkv, hi - lo, group, dim).transpose(0, 1).reshape(hi - lo, hq, dim).to(q.dtype)
        at += new
    return out


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    new, lens = _ints(case["new"]), _ints(case["lens"])
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    cached = 2 * hkv * (2 * dim if case["kind"] == "bf16" else dim + 1)      # a token's keys and values as the cache holds them
    packed = 2 * hkv * 2 * dim
    if case["op"] == "attend":
        keys = sum(n for m, n in zip(new, lens) if m)
        pairs = sum(m * (n - m) + m * (m + 1) // 2 for m, n in zip(new, lens))
        return {"bytes": keys * cached + 2 * sum(new) * hq * dim * 2, "flops": 4 * hq * dim * pairs}
    each = {"write": packed + cached, "store": 2 * packed + 2 * cached, "read": cached + packed}[case["op"]]
    return {"bytes": sum(new) * each, "flops": sum(new) * 2 * hkv * dim}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------
def _exact_values(codes, scale):
    """What bytes of sign, four bits of exponent and three of mantissa stand for, times their row's power of two."""
    bits = codes.view(torch.uint8).long()
    e, m = (bits >> 3) & 15, (bits & 7).double()
    value = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2((e - 10).double())) * (1 - 2 * (bits >> 7)).double()
    return value * torch.exp2(scale.view(torch.uint8).double() - 127)[..., None]


def _exact_rounded(x):
    """x in 64 bits, each row to multiples of what e4m3 resolves under the row's power of two; ties to even."""
    top = x.abs().amax(-1, keepdim=True)
    power = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 448)).clamp(min=SMALLEST))
    # (the logarithm may miss a border by its rounding)
    power = torch.where(top > 448 * power, 2 * power, power)
    power = torch.where((top <= 224 * power) & (power > 2.0 ** SMALLEST), power / 2, power)
    y = (x / power).abs()
    step = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6)))) / 8
    return torch.sign(x) * torch.round(y / step) * step * power


def exact(case, seed):
    s = prepare(case, seed)
    new, lens, page = s["new"], s["lens"], case["page"]
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    tables = s["table"].tolist()

    def cached(name, i, lo, hi):
        """Keys or values of request i at positions lo to hi: (kv heads, hi - lo, dim)."""
        first, last = lo // page, (hi + page - 1) // page
        index = torch.tensor(tables[i][first:last], device=DEV)
        part = s[name + "_pages"].view(torch.uint8 if case["kind"] == "e4m3" else torch.bfloat16)[index]
        part = part.double() if case["kind"] == "bf16" else _exact_values(part, s[name + "_scale"].view(torch.uint8)[index])
        return part.permute(1, 0, 2, 3).flatten(1, 2)[:, lo - first * page:hi - first * page]

    if case["op"] == "read":
        return tuple(torch.cat([cached(name, i, n - m, n).transpose(0, 1) for i, (m, n) in enumerate(zip(new, lens)) if m]) for name in ("k", "v"))
    if case["op"] == "store":
        return tuple(_exact_rounded(s[name].double()) for name in ("k", "v"))
    if case["op"] == "write":
        out = []
        for name in ("k", "v"):
            pages, at = s[name + "_pages"].double(), 0
            for i, (m, n) in enumerate(zip(new, lens)):
                where = torch.arange(n - m, n, device=DEV)
                pages[s["table"][i].long()[where // page], :, where % page] = s[name][at:at + m].double()
                at += m
            out.append(pages)
        return tuple(out)
    out, group = [], hq // hkv
    for i, (q, n) in enumerate(zip(s["q"].double().split(new), lens)):
        m = q.shape[0]
        if m == 0:
            continue
        k, v = cached("k", i, 0, n), cached("v", i, 0, n)
        o = torch.empty_like(q)
        for lo in range(0, m, 256):
            part = q[lo:lo + 256]
            seen = torch.arange(n, device=DEV)[None] <= (n - m + lo + torch.arange(part.shape[0], device=DEV))[:, None]
            for h in range(hq):
                logits = (part[:, h] @ k[h // group].T / math.sqrt(dim)).masked_fill(~seen, -math.inf)
                o[lo:lo + 256, h] = torch.softmax(logits, -1) @ v[h // group]
            o[lo:lo + 256][~seen.any(-1)] = 0
        out.append(o)
    return torch.cat(out)
