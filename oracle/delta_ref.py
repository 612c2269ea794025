"""CPU restatements of a gated-delta-rule layer's operators in 64 bits, written token by token from their definitions; autograd gives their gradients."""
import torch


def gates(a, b, a_log, dt_bias):
    """Decay factor and write strength of every row and head."""
    return torch.exp(-torch.exp(a_log) * torch.nn.functional.softplus(a + dt_bias, threshold=60)), torch.sigmoid(b)


def unit(x):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6)


def gated_delta_rule(q, k, v, a, b, a_log, dt_bias, lens, initial=None, scale=None, l2_norm=True):
    """q, k (T, Hk, Dk), v (T, Hv, Dv), a, b (T, Hv) in double -> o (T, Hv, Dv), states (N, Hv, Dk, Dv)."""
    rep = v.shape[1] // q.shape[1]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    if l2_norm:
        q, k = unit(q), unit(k)
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    decay, beta = gates(a, b, a_log, dt_bias)
    outs, states, t = [], [], 0
    for n, length in enumerate(lens):
        s = initial[n] if initial is not None else torch.zeros(v.shape[1], q.shape[2], v.shape[2], dtype=q.dtype)
        for _ in range(length):
            s = s * decay[t][:, None, None]
            miss = v[t] - (s * k[t][:, :, None]).sum(1)
            s = s + k[t][:, :, None] * (beta[t][:, None] * miss)[:, None, :]
            outs.append(scale * (s * q[t][:, :, None]).sum(1))
            t += 1
        states.append(s)
    return torch.stack(outs) if outs else v[:0], torch.stack(states)


def short_conv(x, weight, bias, lens, initial=None, silu=True):
    """x (T, C), weight (C, W) -> y (T, C), the last W - 1 inputs of every sequence (N, C, W - 1)."""
    width, outs, states, t = weight.shape[1], [], [], 0
    for n, length in enumerate(lens):
        before = initial[n].t() if initial is not None else torch.zeros(width - 1, x.shape[1], dtype=x.dtype)
        seen = torch.cat([before, x[t:t + length]])
        t += length
        z = sum(seen[j:j + length] * weight[:, j] for j in range(width))
        z = z if bias is None else z + bias
        outs.append(z * torch.sigmoid(z) if silu else z)
        states.append(seen[seen.shape[0] - (width - 1):].t())
    return torch.cat(outs), torch.stack(states)


def rms_norm(x, weight, eps=1e-6, offset=False):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (weight + 1 if offset else weight)


def gated_rms_norm(x, gate, weight, eps=1e-6, offset=False):
    return rms_norm(x, weight, eps, offset) * gate * torch.sigmoid(gate)


def residual_rms_norm(x, y, weight, post=None, gate=None, scale=None, eps=1e-6, offset=False):
    part = y if post is None else rms_norm(y, post, eps, offset)
    part = part if gate is None else part * torch.sigmoid(gate)
    part = part if scale is None else part * scale
    return x + part, rms_norm(x + part, weight, eps, offset)
