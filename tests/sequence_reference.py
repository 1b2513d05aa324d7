"""The sequence operators from their definitions, in 64 bits (torch, any device)."""
import math

import torch

TYPES = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}


def layer_norm(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1)
    centred = x - mean[:, None]
    rstd = 1 / torch.sqrt((centred * centred).mean(-1) + eps)
    y = centred * rstd[:, None]
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, mean, rstd


def layer_norm_grad(x, w, mean, rstd, dy):
    x, dy = x.double(), dy.double()
    xhat = (x - mean.double()[:, None]) * rstd.double()[:, None]
    g = dy if w is None else dy * w.double()
    dx = rstd.double()[:, None] * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return dx, (dy * xhat).sum(0), dy.sum(0)


def _weights(log_decay, n, device):
    """l^(i - j) for j <= i, else 0; l^0 = 1 for every l."""
    i = torch.arange(n, device=device)
    gap = (i[:, None] - i[None, :]).double()
    w = torch.where(gap == 0, 1.0, torch.exp(gap * log_decay))
    return torch.where(gap < 0, 0.0, w)


def power(log_decay, n):
    """l^n for a tensor of exponents n >= 0."""
    return torch.where(n == 0, 1.0, torch.exp(n.double() * log_decay))


def attention(q, k, v, log_decay, scale, s0=None):
    """One sequence: q [T, H, Dk], k [T, G, Dk], v [T, G, Dv], s0 [H, Dk, Dv] -> o [T, H, Dv], state."""
    n, heads, _ = q.shape
    share = heads // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    o = torch.empty(n, heads, v.shape[2], dtype=torch.float64, device=q.device)
    state = torch.zeros(heads, q.shape[2], v.shape[2], dtype=torch.float64, device=q.device)
    at = torch.arange(n, device=q.device)
    for h in range(heads):
        g, kh, vh = log_decay[h].double(), k[:, h // share], v[:, h // share]
        o[:, h] = ((q[:, h] @ kh.T) * _weights(g, n, q.device)) @ vh
        state[h] = (kh * power(g, n - 1 - at)[:, None]).T @ vh
        if s0 is not None:
            o[:, h] += power(g, at + 1)[:, None] * (q[:, h] @ s0[h].double())
            state[h] += power(g, torch.tensor(n, device=q.device)) * s0[h].double()
    return scale * o, state


def attention_grad(q, k, v, log_decay, scale, do, s0=None, ds=None):
    n, heads, _ = q.shape
    share = heads // k.shape[1]
    q, k, v, do = (t.double() for t in (q, k, v, do))
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    ds0 = torch.zeros(heads, q.shape[2], v.shape[2], dtype=torch.float64, device=q.device)
    at = torch.arange(n, device=q.device)
    for h in range(heads):
        g, kh, vh = log_decay[h].double(), k[:, h // share], v[:, h // share]
        w = scale * _weights(g, n, q.device)
        seen, back = w * (q[:, h] @ kh.T), w * (do[:, h] @ vh.T)
        dq[:, h] = back @ kh
        dk[:, h // share] += back.T @ q[:, h]
        dv[:, h // share] += seen.T @ do[:, h]
        ds0[h] = scale * (q[:, h] * power(g, at + 1)[:, None]).T @ do[:, h]
        if s0 is not None:
            dq[:, h] += scale * power(g, at + 1)[:, None] * (do[:, h] @ s0[h].double().T)
        if ds is not None:
            late = power(g, n - 1 - at)[:, None]
            dk[:, h // share] += late * (vh @ ds[h].double().T)
            dv[:, h // share] += late * (kh @ ds[h].double())
            ds0[h] += power(g, torch.tensor(n, device=q.device)) * ds[h].double()
    return dq, dk, dv, ds0


def rel(got, want):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isfinite(got), torch.isfinite(want))
    d, n = torch.linalg.vector_norm(got - want), torch.linalg.vector_norm(want)
    return float(d / n) if float(n) else float(d)


def norm_tolerance(dtype, features):
    """A result's own rounding (half a unit: 2^-24, 2^-11, 2^-8 of it at most) and f32 arithmetic before it:
    a sum of n terms held in at least 32 partial sums, some ten further roundings."""
    unit = {"F32": 2.0 ** -24, "F16": 2.0 ** -11, "BF16": 2.0 ** -8}[dtype]
    return unit + 2.0 ** -24 * (16 + math.sqrt(features))


def attention_tolerance(dtype, tokens):
    """Relative 2-norm.  f32: every token rounds the state once (a random walk: sqrt(tokens) units of 2^-24, times
    four for the sums over keys and tokens and the powers of the decay), and 32 units for products split into
    two 11-bit parts.  16-bit types: up to three independent roundings to the type (scores, state, result), each of at
    most half a unit, evenly spread (1 / sqrt(3)): together half a unit."""
    f32 = 2.0 ** -24 * (32 + 4 * math.sqrt(tokens))
    return f32 + {"F32": 0.0, "F16": 2.0 ** -11, "BF16": 2.0 ** -8}[dtype]
