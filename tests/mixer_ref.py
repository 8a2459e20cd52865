"""The token mixers from their definitions, in 64 bits, and the distances their kernels may be off."""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step


def axes_of(rotary, sections, interleaved):
    """Axis of each rotated pair, from the header's words."""
    s = list(sections) + [0] * (3 - len(sections))
    out = []
    for i in range(rotary // 2):
        if interleaved:
            out.append(1 if i % 3 == 1 and i < 3 * s[1] else 2 if i % 3 == 2 and i < 3 * s[2] else 0)
        else:
            out.append(0 if i < s[0] else 1 if i < s[0] + s[1] else 2)
    return out


def rotate(x, pos, rotary, theta, axes):
    """x [T, heads, dim], pos [3 or 1, T] -> (rotated, how far it may be off before its rounding)."""
    x = x.double().cpu()
    y, off = x.clone(), torch.zeros_like(x)
    half = rotary // 2
    for i in range(half):
        angle = pos[axes[i] if pos.shape[0] > 1 else 0].double().cpu() * theta ** (-2.0 * i / rotary)
        c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        a, b = x[..., i], x[..., i + half]
        y[..., i], y[..., i + half] = a * c - b * s, b * c + a * s
        # the angle's 32-bit fraction of a turn, the sine's and cosine's last places and the two products
        # are off by a few 2^-24 of |a| + |b|
        off[..., i] = off[..., i + half] = (a.abs() + b.abs()) * 2.0 ** -21
    return y, off


def attend(q, k, v, place, scale):
    """q [rows, dim] of one head, k and v [keys, dim], place [rows]: position of each row (-1 and less: none).
    -> (out, how far 32-bit arithmetic with probabilities in q's type may be off), float64."""
    dt, dim = q.dtype, q.shape[1]
    u, big = U[dt], k.shape[0]
    q, k, v = q.double(), k.double(), v.double()
    if big == 0:
        z = torch.zeros_like(q)
        return z, z.clone()
    seen = torch.arange(big, device=q.device) <= place[:, None]
    s = (q @ k.T) * scale
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = p.sum(-1, keepdim=True)
    div = torch.where(total == 0, 1.0, total)
    o, size = p @ v / div, p @ v.abs() / div
    # a score is a sum of dim products in 32 bits; a probability takes the score's error twice (its own and in the sum),
    # the exponential's, and one rounding to the type (below 2^-14 fp16 has fixed steps of 2^-24)
    ds = dim * 2.0 ** -24 * scale * ((q.abs() @ k.abs().T) * seen).amax(-1, keepdim=True)
    off = u * o.abs() + (u + 2 * ds + 2.0 ** -18) * size + 1e-7
    if dt == torch.float16:
        off += 2.0 ** -25 * (seen.double() @ v.abs()) / div
    return o, off


def attend_batch(q, kc, vc, table, kv_len, cu, scale, page):
    """All sequences and heads: q [T, hq, dim] -> out, off [T, hq, dim] (nan where no sequence has a row)."""
    T, hq, dim = q.shape
    hkv = kc.shape[1]
    out = torch.full((T, hq, dim), math.nan, dtype=torch.float64, device=q.device)
    off = torch.zeros_like(out)
    for i, n in enumerate(kv_len):
        a, b = cu[i], cu[i + 1]
        if a == b:
            continue
        pages = table[i, : -(-n // page)].long()
        place = torch.arange(n - (b - a), n, device=q.device)
        for h in range(hq):
            k, v = (c[pages, h // (hq // hkv)].reshape(-1, dim)[:n] for c in (kc, vc))
            out[a:b, h], off[a:b, h] = attend(q[a:b, h], k, v, place, scale)
    return out, off


def delta(q, k, v, g, beta, S, l2norm, scale):
    """One sequence, all value heads: the recurrence as it is defined.  S [hv, dk, dv] -> out [T, hv, dv], S."""
    hv = v.shape[1]
    group = hv // q.shape[1]
    q, k, v, g, beta, S = (x.double() for x in (q, k, v, g, beta, S))
    if l2norm:
        q = q / torch.sqrt(q.pow(2).sum(-1, keepdim=True) + 1e-6)
        k = k / torch.sqrt(k.pow(2).sum(-1, keepdim=True) + 1e-6)
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    out = torch.zeros_like(v)
    for t in range(v.shape[0]):
        S = S * torch.exp(g[t])[:, None, None]
        u = beta[t][:, None] * (v[t] - (k[t][:, :, None] * S).sum(1))
        S = S + k[t][:, :, None] * u[:, None, :]
        out[t] = scale * (q[t][:, :, None] * S).sum(1)
    return out, S


def rel(x, y):
    return float((x.double() - y.double()).norm() / y.double().norm().clamp(min=1e-300))
