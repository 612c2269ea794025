"""The operators of a gated-delta-rule layer and of the norms around a block: their calls, and the same in elementary torch operations.

``op`` names the operator, ``mode`` the direction:

* ``delta``  ``gated_delta_rule``: ``train`` (forward and backward, every gradient), ``prefill`` (no graph, from a state to a state);
             ``gated_delta_step``: ``step`` (one token for each of ``batch`` requests, the state updated in place)
* ``conv``   ``short_conv`` with ``train``; ``short_conv_step`` with ``step``
* ``gnorm``  ``gated_rms_norm``, the norm behind the rule with its SiLU gate: ``train``, ``forward``
* ``rnorm``  ``residual_rms_norm``, residual add and the next block's norm: ``train``, ``forward``; ``post`` a norm of the block's output
             in front of the addition, ``gate`` a sigmoid gate on it, ``scale`` a scale per channel, ``stream`` the residual's type

``segments`` holds the lengths of the packed sequences, comma-separated.
"""
import math

import torch
import torch.nn.functional as F

own = False
DEV = "cuda"
CHUNK = 64
EPS = 1e-6


# ---- cases ----------------------------------------------------------------------------------------------------------
def _delta(mode, segments, hk, hv, dk=128, dv=128, **more):
    return dict(op="delta", mode=mode, segments=segments, hk=hk, hv=hv, dk=dk, dv=dv, **more)


#: the packed hybrid-stack batch (configuration C5): 16 384 tokens
PACKED = ("716,65,73,107,133,129,75,135,512,1379,214,227,270,675,972,1669,234,740,208,1112,141,1309,367,789,407,190,354,76,74,400,333,1147,1152")


def listed():
    return [
        # one request's next token in one layer: the smallest call, all latency
        dict(name="delta_step_1", op="delta", mode="step", batch=1, hk=16, hv=32, dk=128, dv=128),
        # a serving batch's next tokens: the states pass through memory once
        dict(name="delta_step_256", op="delta", mode="step", batch=256, hk=16, hv=32, dk=128, dv=128),
        # prompts of four requests, one a single token and one continued from a state
        dict(_delta("prefill", "4000,1,63,700", 16, 32), name="delta_prefill_5k"),
        # odd heads, rows and lengths, an empty sequence: a small model's unpadded batch
        dict(_delta("train", "1,130,0,65,333,64,7", 3, 6, 64, 96), name="delta_train_odd"),
        # a training step on the packed hybrid-stack batch
        dict(_delta("train", PACKED, 16, 32), name="delta_train_16k"),
        # a training step on one long document: few sequences, a long way from the first chunk to the last
        dict(_delta("train", "32768", 16, 32), name="delta_train_32k"),
        # the convolution in front of the rule, over its q, k and v channels, same batch
        dict(name="conv_train_16k", op="conv", mode="train", segments=PACKED, channels=8192, width=4, bias=False),
        dict(name="conv_step_256", op="conv", mode="step", batch=256, channels=8192, width=4, bias=False),
        # the norm behind the rule: a training step, and a decoding batch
        dict(name="gnorm_train_16k", op="gnorm", mode="train", tokens=16384, heads=32, dim=128),
        dict(name="gnorm_step_256", op="gnorm", mode="forward", tokens=256, heads=32, dim=128),
        # residual add and the next block's norm: a training step of an 8-billion-parameter width, plain
        dict(name="rnorm_train_8k", op="rnorm", mode="train", tokens=8192, width=4096, post=False, gate=False, scale=False, stream="bf16"),
        # all of it at once, an odd number of rows, the residual stream in 32 bits
        dict(name="rnorm_gated_1k", op="rnorm", mode="train", tokens=1037, width=2560, post=True, gate=True, scale=True, stream="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _lengths(rng, total, most):
    """``total`` tokens cut into up to ``most`` sequences at random places (equal places leave empty ones), four tokens each at the mean."""
    n = _log(rng, 1, min(most, total // 4))
    cuts = sorted(rng.randint(0, total) for _ in range(n - 1))
    return ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [total]))


def draw(rng):
    op, mode = rng.choice([("delta", "train"), ("delta", "train"), ("delta", "prefill"), ("delta", "step"), ("conv", "train"), ("conv", "step"),
                           ("gnorm", "train"), ("gnorm", "forward"), ("rnorm", "train"), ("rnorm", "forward")])
    if op == "delta":
        hk = rng.choice([1, 2, 3, 4, 8, 16])
        hv = hk * rng.choice([1, 2, 2, 3, 4])
        dk, dv = rng.choice([(128, 128), (128, 128), (64, 64), (64, 128), (96, 120), (40, 72)])
        if mode == "step":
            return dict(op=op, mode=mode, batch=_log(rng, 1, 8192 // hv), hk=hk, hv=hv, dk=dk, dv=dv)
        return _delta(mode, _lengths(rng, _log(rng, 16, min(20000, 500000 // hv)), 40), hk, hv, dk, dv)
    if op == "conv":
        channels, width, bias = 8 * _log(rng, 8, 1024), rng.choice([2, 3, 4, 4]), rng.random() < 0.5
        if mode == "step":
            return dict(op=op, mode=mode, batch=_log(rng, 1, 1024), channels=channels, width=width, bias=bias)
        return dict(op=op, mode=mode, segments=_lengths(rng, _log(rng, 16, min(60000, 130000000 // channels)), 40), channels=channels, width=width, bias=bias)
    if op == "gnorm":
        heads, dim = rng.choice([1, 4, 6, 16, 32]), rng.choice([64, 128, 128, 256, 72])
        return dict(op=op, mode=mode, tokens=_log(rng, 1, 60000000 // (heads * dim) + 1), heads=heads, dim=dim)
    width = 8 * _log(rng, 8, 1024)
    return dict(op=op, mode=mode, tokens=_log(rng, 1, min(30000, 40000000 // width)), width=width, post=rng.random() < 0.5, gate=rng.random() < 0.5,
                scale=rng.random() < 0.5, stream=rng.choice(["bf16", "bf16", "fp32"]))


def _lens(case):
    return [int(n) for n in case["segments"].split(",")]


# ---- inputs ---------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    bf = torch.bfloat16

    def rn(*shape, std=1.0, dtype=bf, mean=0.0):
        return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(dtype)

    def leaf(t):
        return t.requires_grad_(True) if case["mode"] == "train" else t

    s = {"case": dict(case)}
    if case["op"] == "delta":
        hk, hv, dk, dv = (case[x] for x in ("hk", "hv", "dk", "dv"))
        rows = case["batch"] if case["mode"] == "step" else sum(_lens(case))
        # q, k and v lie side by side in one tensor, as the convolution leaves them, and are read in place
        mixed = F.silu(rn(rows, 2 * hk * dk + hv * dv, dtype=torch.float32)).to(bf)
        s["q"] = leaf(mixed[:, :hk * dk].unflatten(1, (hk, dk)))
        s["k"] = leaf(mixed[:, hk * dk:2 * hk * dk].unflatten(1, (hk, dk)))
        s["v"] = leaf(mixed[:, 2 * hk * dk:].unflatten(1, (hv, dv)))
        s["a"], s["b"] = leaf(rn(rows, hv)), leaf(rn(rows, hv))
        # decay rates and time steps as such layers start out: rates 1 to 16, steps 0.001 to 0.1
        u = torch.rand(2, hv, generator=g, device=DEV)
        step = torch.exp(u[1] * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
        s["a_log"] = leaf(torch.log(1 + 15 * u[0]).to(bf))
        s["dt_bias"] = leaf((step + torch.log(-torch.expm1(-step))).to(bf))
        if case["mode"] == "step":
            s["state"] = rn(rows, hv, dk, dv, std=0.1, dtype=torch.float32)
        else:
            lens = _lens(case)
            s["cu"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
            if case["mode"] == "prefill":
                s["state"] = rn(len(lens), hv, dk, dv, std=0.1, dtype=torch.float32)
            else:
                s["grad"] = rn(rows, hv, dv)
    elif case["op"] == "conv":
        c, w = case["channels"], case["width"]
        rows = case["batch"] if case["mode"] == "step" else sum(_lens(case))
        s["x"] = leaf(rn(rows, c))
        s["weight"] = leaf(rn(c, w, std=w ** -0.5))
        s["bias"] = leaf(rn(c, std=0.1)) if case["bias"] else None
        if case["mode"] == "step":
            s["state"] = rn(rows, c, w - 1)
        else:
            lens = _lens(case)
            s["cu"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
            s["grad"] = rn(rows, c)
    elif case["op"] == "gnorm":
        t, h, d = case["tokens"], case["heads"], case["dim"]
        s["x"], s["z"], s["weight"] = leaf(rn(t, h, d, std=0.5)), leaf(rn(t, h, d)), leaf(rn(d, std=0.1, mean=1.0))
        s["grad"] = rn(t, h, d) if case["mode"] == "train" else None
    else:
        t, c = case["tokens"], case["width"]
        s["x"] = leaf(rn(t, c, std=2.0, dtype=bf if case["stream"] == "bf16" else torch.float32))
        s["y"], s["weight"] = leaf(rn(t, c)), leaf(rn(c, std=0.1, mean=1.0))
        s["post"] = leaf(rn(c, std=0.1, mean=1.0)) if case["post"] else None
        s["gate"] = leaf(rn(t, c)) if case["gate"] else None
        s["scale"] = leaf(rn(c, std=0.1, mean=0.5)) if case["scale"] else None
        if case["mode"] == "train":
            s["grads"] = (rn(t, c, dtype=s["x"].dtype), rn(t, c))
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def _grads(outs, grads, leaves):
    """The outputs and the gradient of every leaf that is there."""
    names = [n for n, t in leaves.items() if t is not None]
    got = torch.autograd.grad(outs, [leaves[n] for n in names], grads)
    return {"d" + n: t for n, t in zip(names, got)}


def run(s):
    case = s["case"]
    if own:
        import vlm_training_amd as V
        delta, delta_step, conv, conv_step, gnorm, rnorm = (V.gated_delta_rule, V.gated_delta_step, V.short_conv, V.short_conv_step, V.gated_rms_norm,
                                                            V.residual_rms_norm)
    else:
        delta, delta_step, conv, conv_step, gnorm, rnorm = _plain_delta, _plain_delta_step, _plain_conv, _plain_conv_step, _plain_gnorm, _plain_rnorm
    if case["op"] == "delta":
        names = ("q", "k", "v", "a", "b", "a_log", "dt_bias")
        args = [s[n] for n in names]
        if case["mode"] == "step":
            return {"o": delta_step(*args, s["state"]), "state": s["state"]}
        if case["mode"] == "prefill":
            with torch.no_grad():
                o, state = delta(*args, s["cu"], initial_state=s["state"], return_final_state=True)
            return {"o": o, "state": state}
        o = delta(*args, s["cu"])
        return {"o": o.detach(), **_grads([o], [s["grad"]], {n: s[n] for n in names})}
    if case["op"] == "conv":
        if case["mode"] == "step":
            return {"y": conv_step(s["x"], s["state"], s["weight"], s["bias"]), "state": s["state"]}
        y = conv(s["x"], s["weight"], s["bias"], s["cu"])
        return {"y": y.detach(), **_grads([y], [s["grad"]], {n: s[n] for n in ("x", "weight", "bias")})}
    if case["op"] == "gnorm":
        y = gnorm(s["x"], s["z"], s["weight"])
        return {"y": y.detach(), **(_grads([y], [s["grad"]], {n: s[n] for n in ("x", "z", "weight")}) if case["mode"] == "train" else {})}
    x, h = rnorm(s["x"], s["y"], s["weight"], post_weight=s["post"], gate=s["gate"], scale=s["scale"])
    out = {"x": x.detach(), "h": h.detach()}
    if case["mode"] == "train":
        out.update(_grads([x, h], list(s["grads"]), {n: s[n] for n in ("x", "y", "weight", "post", "gate", "scale")}))
    return out


# ---- the plain forms: 32 bits throughout, rounded at the end ---------------------------------------------------------
def _unit(x):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS)


def _gates(a, b, a_log, dt_bias):
    return -torch.exp(a_log.float()) * F.softplus(a.float() + dt_bias.float()), torch.sigmoid(b.float())


def _unit_lower_inverse(m):
    """Inverse of I + strictly lower m (..., 64, 64): of the diagonal blocks of 1, 2, 4 .. rows in turn,
    [[A, 0], [C, B]]^-1 = [[A^-1, 0], [-B^-1 C A^-1, B^-1]]."""
    lead, n, size = m.shape[:-2], m.shape[-1], 1
    inv = torch.ones(*lead, n, 1, 1, dtype=m.dtype, device=m.device)
    while size < n:
        blocks = m.unflatten(-2, (n // (2 * size), 2, size)).unflatten(-1, (n // (2 * size), 2, size))
        c = torch.stack([blocks[..., i, 1, :, i, 0, :] for i in range(n // (2 * size))], dim=-3)
        pair = inv.unflatten(-3, (n // (2 * size), 2))
        a, b = pair[..., 0, :, :], pair[..., 1, :, :]
        low = -(b @ c @ a)
        inv = torch.cat([torch.cat([a, torch.zeros_like(a)], -1), torch.cat([low, b], -1)], -2)
        size *= 2
    return inv[..., 0, :, :]


def _plain_delta(q, k, v, a, b, a_log, dt_bias, cu, initial_state=None, return_final_state=False):
    lens = (cu[1:] - cu[:-1]).tolist()
    rows, hk, dk, hv, dv = q.shape[0], q.shape[1], q.shape[2], v.shape[1], v.shape[2]
    starts = [sum(lens[:i]) for i in range(len(lens))]
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    # chunk c of every sequence that has one, the long ones first: a table of row numbers, padded with one more (zero) row
    table, counts = [], []
    for c in range((max(lens) + CHUNK - 1) // CHUNK):
        live = [i for i in order if lens[i] > c * CHUNK]
        counts.append(len(live))
        table += [[starts[i] + c * CHUNK, min(CHUNK, lens[i] - c * CHUNK)] for i in live]
    first, size = torch.tensor(table, dtype=torch.int64).reshape(-1, 2).to(q.device, non_blocking=True).unbind(1)
    at = torch.arange(CHUNK, device=q.device)
    index = torch.where(at < size[:, None], first[:, None] + at, rows)                     # (chunks, 64)

    def chunks(x):                                                                          # (rows, H, ..) -> (chunks, H, 64, ..)
        return torch.cat([x, torch.zeros_like(x[:1]) if rows else x.new_zeros(1, *x.shape[1:])])[index].transpose(1, 2)

    g, beta = _gates(a, b, a_log, dt_bias)
    rep = hv // hk
    qc = chunks(_unit(q.float()).repeat_interleave(rep, 1)) * dk ** -0.5
    kc, vc, gc, bc = chunks(_unit(k.float()).repeat_interleave(rep, 1)), chunks(v.float()), chunks(g), chunks(beta)[..., None]
    big = gc.double().cumsum(-1)
    diff = (big[..., :, None] - big[..., None, :]).float()
    lower = at[:, None] >= at
    decay = torch.exp(torch.where(lower, diff, 0.0)) * lower
    inv = _unit_lower_inverse(bc * (kc @ kc.mT) * decay * (at[:, None] > at))
    attn = (qc @ kc.mT) * decay
    grow, left, whole = torch.exp(big)[..., None].float(), torch.exp(big[..., -1:] - big)[..., None].float(), torch.exp(big[..., -1])[..., None, None].float()
    u, w, qs, ks = inv @ (bc * vc), inv @ (bc * grow * kc), qc * grow, kc * left
    state = (initial_state if initial_state is not None else torch.zeros(len(lens), hv, dk, dv, device=q.device))[order]
    outs, done = [], []
    for n, *x in zip(counts, *(t.split(counts) for t in (u, w, qs, ks, attn, whole))):
        un, wn, qn, kn, pn, en = x
        done.append(state[n:])
        state = state[:n]
        new = un - wn @ state
        outs.append(qn @ state + pn @ new)
        state = en * state + kn.mT @ new
    out = torch.cat(outs).transpose(1, 2).reshape(-1, hv, dv)
    o = torch.zeros(rows + 1, hv, dv, device=q.device).index_copy(0, index.reshape(-1), out)[:rows].to(v.dtype)
    if not return_final_state:
        return o
    back = torch.empty(len(order), dtype=torch.int64)
    back[torch.tensor(order)] = torch.arange(len(order))
    return o, torch.cat([state, *reversed(done)])[back.to(q.device)]


def _plain_delta_step(q, k, v, a, b, a_log, dt_bias, state):
    g, beta = _gates(a, b, a_log, dt_bias)
    rep = v.shape[1] // q.shape[1]
    qf, kf = (_unit(x.float()).repeat_interleave(rep, 1)[..., None] for x in (q, k))       # (B, H, Dk, 1)
    state *= torch.exp(g)[..., None, None]
    new = beta[..., None] * (v.float() - (kf * state).sum(-2))
    state += kf * new[..., None, :]
    return ((qf * state).sum(-2) * q.shape[-1] ** -0.5).to(v.dtype)


def _plain_conv(x, weight, bias, cu):
    rows, width = x.shape[0], weight.shape[1]
    at = torch.arange(rows, device=x.device)
    first = cu.long()[torch.searchsorted(cu[1:].contiguous(), at.int(), right=True)]
    xf, w = x.float(), weight.float()
    z = sum((torch.where((at - back >= first)[:, None], F.pad(xf, (0, 0, back, 0))[:rows], 0.0) * w[:, width - 1 - back] for back in range(width)),
            bias.float() if bias is not None else 0.0)
    return (z * torch.sigmoid(z)).to(x.dtype)


def _plain_conv_step(x, state, weight, bias):
    past = torch.cat([state, x[..., None]], -1)
    z = (past.float() * weight.float()).sum(-1) + (bias.float() if bias is not None else 0.0)
    state.copy_(past[..., 1:])
    return (z * torch.sigmoid(z)).to(x.dtype)


def _norm(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()


def _plain_gnorm(x, z, weight):
    zf = z.float()
    return (_norm(x.float(), weight) * zf * torch.sigmoid(zf)).to(x.dtype)


def _plain_rnorm(x, y, weight, post_weight=None, gate=None, scale=None):
    part = y.float() if post_weight is None else _norm(y.float(), post_weight)
    if gate is not None:
        part = part * torch.sigmoid(gate.float())
    if scale is not None:
        part = part * scale.float()
    new = x.float() + part
    return new.to(x.dtype), _norm(new, weight).to(y.dtype)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "delta":
        hk, hv, dk, dv = (case[x] for x in ("hk", "hv", "dk", "dv"))
        rows = case["batch"] if case["mode"] == "step" else sum(_lens(case))
        inputs, cell, state = rows * (2 * (2 * hk * dk + hv * dv) + 4 * hv), rows * hv * dk * dv, 4 * hv * dk * dv
        if case["mode"] == "step":
            return {"bytes": inputs + rows * 2 * hv * dv + 2 * rows * state, "flops": 7 * cell}
        if case["mode"] == "prefill":
            return {"bytes": inputs + rows * 2 * hv * dv + 2 * len(_lens(case)) * state, "flops": 7 * cell}
        # the forward reads the inputs and writes o; the backward reads them and dO and writes a gradient for each
        return {"bytes": 3 * inputs + 2 * rows * 2 * hv * dv, "flops": 21 * cell}
    if case["op"] == "conv":
        c, w = case["channels"], case["width"]
        if case["mode"] == "step":
            return {"bytes": case["batch"] * c * 2 * (2 + 2 * (w - 1)) + 2 * c * w, "flops": 2 * case["batch"] * c * w}
        rows = sum(_lens(case))
        return {"bytes": rows * c * 2 * 5 + 4 * c * w, "flops": 6 * rows * c * w}
    if case["op"] == "gnorm":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * (3 if case["mode"] == "forward" else 8), "flops": n * (8 if case["mode"] == "forward" else 30)}
    n, e = case["tokens"] * case["width"], 2 if case["stream"] == "bf16" else 4
    forward = n * (2 * e + 4 + 2 * case["gate"])
    # the backward reads x', both gradients, and y and the gate where something depends on them; it writes dx, dy and dgate
    backward = n * (3 * e + 2 + 2 + 2 * (case["post"] or case["gate"] or case["scale"]) + 4 * case["gate"])
    return {"bytes": forward + (backward if case["mode"] == "train" else 0), "flops": n * (10 if case["mode"] == "forward" else 40)}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "delta" and case["mode"] != "step":
        lens = _lens(case)
        if max(lens) * (45 * 6e-6 + len(lens) * case["hv"] * case["dk"] * case["dv"] * 8 * 40 / 3e12) > 18:
            return None
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"delta": _exact_delta, "conv": _exact_conv, "gnorm": _exact_gnorm, "rnorm": _exact_rnorm}[case["op"]](case, s)


def _wide(s, names):
    return {n: s[n].detach().double().requires_grad_(True) for n in names if s[n] is not None}


def _exact_delta(case, s):
    names = ("q", "k", "v", "a", "b", "a_log", "dt_bias")
    x = _wide(s, names)
    rep, scale = case["hv"] // case["hk"], case["dk"] ** -0.5
    q = (x["q"] / torch.sqrt((x["q"] ** 2).sum(-1, keepdim=True) + EPS)).repeat_interleave(rep, 1)
    k = (x["k"] / torch.sqrt((x["k"] ** 2).sum(-1, keepdim=True) + EPS)).repeat_interleave(rep, 1)
    alpha = torch.exp(-torch.exp(x["a_log"]) * torch.log1p(torch.exp(x["a"] + x["dt_bias"])))
    beta = 1 / (1 + torch.exp(-x["b"]))
    parts = [t.detach() for t in (q, k, x["v"], alpha, beta)]
    rows = parts[0].shape[0]
    if case["mode"] == "step":
        lens, first = [1] * rows, s["state"].double()
    else:
        lens = _lens(case)
        first = s["state"].double() if case["mode"] == "prefill" else torch.zeros(len(lens), case["hv"], case["dk"], case["dv"], dtype=torch.float64, device=DEV)
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    starts = torch.tensor([sum(lens[:i]) for i in range(len(lens))], device=DEV)[order]
    live = [sum(n > t for n in lens) for t in range(max(lens))]
    state = first[order].clone()
    o = torch.zeros(rows, case["hv"], case["dv"], dtype=torch.float64, device=DEV)

    def token(t, n):
        at = starts[:n] + t
        return (at, *(p[at] for p in parts))

    def forward(state, t, n):
        """The token's state from the one before it, and the value that it adds along k."""
        _, _, kt, vt, at_, bt = token(t, n)
        decayed = state[:n] * at_[..., None, None]
        miss = vt - torch.matmul(kt[..., None, :], decayed).squeeze(-2)
        return decayed, miss, decayed + kt[..., :, None] * (bt[..., None] * miss)[..., None, :]

    keep, every = {}, 64
    for t, n in enumerate(live):
        if t % every == 0:
            keep[t] = state.clone()
        at, qt = token(t, n)[:2]
        state[:n] = forward(state, t, n)[2]
        o[at] = scale * torch.matmul(qt[..., None, :], state[:n]).squeeze(-2)
    back = torch.empty(len(order), dtype=torch.int64)
    back[torch.tensor(order)] = torch.arange(len(order))
    if case["mode"] != "train":
        return {"o": o, "state": state[back.to(DEV)]}
    do, ds = s["grad"].double(), torch.zeros_like(state)
    dq, dk, dv, dalpha, dbeta = (torch.zeros_like(p) for p in parts)
    for t0 in sorted(keep, reverse=True):
        states, here = [], keep[t0]
        for t in range(t0, min(t0 + every, len(live))):
            states.append(here[:live[t]])
            here = forward(here, t, live[t])[2]
        for t in range(min(t0 + every, len(live)) - 1, t0 - 1, -1):
            n, before = live[t], states[t - t0]
            at, qt, kt, _, al, bt = token(t, n)
            decayed, miss, now = forward(before, t, n)
            d = scale * do[at]
            dq[at] = torch.matmul(now, d[..., None]).squeeze(-1)
            grad = ds[:n] + qt[..., :, None] * d[..., None, :]
            dadd = torch.matmul(kt[..., None, :], grad).squeeze(-2)
            dbeta[at] = (dadd * miss).sum(-1)
            dmiss = bt[..., None] * dadd
            dv[at] = dmiss
            dk[at] = torch.matmul(grad, (bt[..., None] * miss)[..., None]).squeeze(-1) - torch.matmul(decayed, dmiss[..., None]).squeeze(-1)
            grad = grad - kt[..., :, None] * dmiss[..., None, :]
            dalpha[at] = (grad * before).sum((-1, -2))
            ds[:n] = grad * al[..., None, None]
    got = torch.autograd.grad([q, k, x["v"], alpha, beta], [x[n] for n in names], [dq, dk, dv, dalpha, dbeta])
    return {"o": o, **{"d" + n: t for n, t in zip(names, got)}}


def _exact_conv(case, s):
    x = _wide(s, ("x", "weight", "bias"))
    width = case["width"]
    if case["mode"] == "step":
        past = torch.cat([s["state"].double(), x["x"][..., None]], -1)
        z = (past * x["weight"]).sum(-1) + x.get("bias", 0.0)
        return {"y": (z / (1 + torch.exp(-z))).detach(), "state": past[..., 1:].detach()}
    padded, where, at = [], [], 0
    for part in x["x"].split(_lens(case)):
        padded += [x["x"].new_zeros(width - 1, case["channels"]), part]
        where.append(torch.arange(part.shape[0], device=DEV) + at + width - 1)
        at += part.shape[0] + width - 1
    padded, where = torch.cat(padded), torch.cat(where)
    z = x.get("bias", 0.0) + torch.zeros_like(x["x"])
    for j in range(width):
        z = z + padded[where - (width - 1) + j] * x["weight"][:, j]
    y = z / (1 + torch.exp(-z))
    return {"y": y.detach(), **_grads([y], [s["grad"].double()], x)}


def _exact_norm(x, weight):
    return x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + EPS) * weight


def _exact_gnorm(case, s):
    x = _wide(s, ("x", "z", "weight"))
    y = _exact_norm(x["x"], x["weight"]) * x["z"] / (1 + torch.exp(-x["z"]))
    return {"y": y.detach(), **(_grads([y], [s["grad"].double()], x) if case["mode"] == "train" else {})}


def _exact_rnorm(case, s):
    x = _wide(s, ("x", "y", "weight", "post", "gate", "scale"))
    part = _exact_norm(x["y"], x["post"]) if case["post"] else x["y"]
    part = part * x.get("scale", 1.0) / (1 + torch.exp(-x["gate"]) if case["gate"] else 1.0)
    new = x["x"] + part
    h = _exact_norm(new, x["weight"])
    out = {"x": new.detach(), "h": h.detach()}
    return {**out, **_grads([new, h], [g.double() for g in s["grads"]], x)} if case["mode"] == "train" else out
