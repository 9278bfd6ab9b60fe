"""The sequence-memory operators from their definitions in float64, step by step, for the tests of their kernels.  Every function also
returns (or can be called for) the sums of the absolute values of the terms, which the rounding bounds of the tests are relative to."""
import math

import torch


def attention(q, k, v, decay, state=None, reset=None, scale=1.0):
    """(out, state behind the last step); [T, M, H, D] inputs of any type, computed in their type."""
    t, m, h, dk = q.shape
    s = torch.zeros(m, h, dk, v.shape[-1], dtype=q.dtype, device=q.device) if state is None else state
    g, zero, out = decay[None, :, None, None], torch.zeros((), dtype=q.dtype, device=q.device), []
    for i in range(t):
        s = s * g
        if reset is not None:
            s = torch.where((reset[i] != 0)[:, None, None, None], zero, s)
        s = s + k[i][..., :, None] * v[i][..., None, :]
        out.append((q[i][..., :, None] * s).sum(-2) * scale)
    return torch.stack(out) if t else q.new_zeros(0, m, h, v.shape[-1]), s


def attention_grad(q, k, v, decay, dout, dstate_out=None, state=None, reset=None, scale=1.0):
    """(dq, dk, dv, dstate) by the two scans of the definition."""
    t, m, h, dk = q.shape
    dv = v.shape[-1]
    g, zero = decay[None, :, None, None], torch.zeros((), dtype=q.dtype, device=q.device)
    s = torch.zeros(m, h, dk, dv, dtype=q.dtype, device=q.device) if state is None else state
    r = torch.zeros_like(s) if dstate_out is None else dstate_out
    dq, dk_, dv_ = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)

    def border(x, i):
        x = x * g
        return x if reset is None else torch.where((reset[i] != 0)[:, None, None, None], zero, x)

    for i in range(t):
        s = border(s, i) + k[i][..., :, None] * v[i][..., None, :]
        dq[i] = (s * dout[i][..., None, :]).sum(-1) * scale
    for i in range(t - 1, -1, -1):
        r = r + q[i][..., :, None] * dout[i][..., None, :] * scale
        dk_[i] = (r * v[i][..., None, :]).sum(-1)
        dv_[i] = (r * k[i][..., :, None]).sum(-2)
        r = border(r, i)
    return dq, dk_, dv_, r


def normed(x, kind, eps):
    c = x if kind == "rms_norm" else x - x.mean(-1, keepdim=True)
    return c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)


def residual_norm(x, f, gate, gate_act, p, kind, post, pre, eps):
    n = normed(f, kind, eps) if post else f
    if p["post_scale"] is not None:
        n = n * p["post_scale"]
    if p["post_bias"] is not None:
        n = n + p["post_bias"]
    if gate_act != "none":
        n = n * (torch.sigmoid(gate) if gate_act == "sigmoid" else gate * torch.sigmoid(gate))
    y = x + (n if p["res_scale"] is None else n * p["res_scale"])
    if not pre:
        return y, None
    h = normed(y, kind, eps)
    if p["pre_scale"] is not None:
        h = h * p["pre_scale"]
    if p["pre_bias"] is not None:
        h = h + p["pre_bias"]
    return y, h


def logprobs(logits, actions, mask, temperature, top):
    """One row at a time."""
    n, width = logits.shape
    logp, entropy, lse = (torch.zeros(n, dtype=torch.float64) for _ in range(3))
    top_logp, top_action = torch.full((n, top), -math.inf, dtype=torch.float64), torch.full((n, top), -1, dtype=torch.int32)
    for i in range(n):
        x = logits[i].double() / temperature
        ok = (x > -math.inf) | x.isnan()
        if mask is not None:
            ok &= mask[i] != 0
        a = int(actions[i])
        if not bool(ok.any()):
            lse[i], entropy[i] = -math.inf, 0.0
            logp[i] = -math.inf if 0 <= a < width else 0.0
            continue
        xs = x[ok]
        bad = bool((xs.isnan() | (xs == math.inf)).any())
        lse[i] = math.nan if bad else torch.logsumexp(xs, 0)
        p = torch.exp(xs - lse[i])
        entropy[i] = -(torch.where(p > 0, p * (xs - lse[i]), torch.zeros_like(p))).sum() if not bad else math.nan
        logp[i] = 0.0 if not 0 <= a < width else (math.nan if bad else x[a] - lse[i] if bool(ok[a]) else -math.inf)
        order = sorted((j for j in range(width) if bool(ok[j]) and not math.isnan(float(x[j]))), key=lambda j: (-float(logits[i, j]), j))[:top]
        for r, j in enumerate(order):
            top_logp[i, r], top_action[i, r] = x[j] - lse[i], j
    return logp, entropy, lse, top_logp, top_action
