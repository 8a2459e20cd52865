"""8-bit caches and norms from their definitions, in 64 bits, and the distances their kernels may be off."""
import math

import torch

import qe_mixer
from mixer_ref import U

MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def values(codes, scale):
    """What codes [..., dim] with scales [...] stand for, in 64 bits."""
    return codes.double() * scale.double()[..., None]


def quantised(x, codes):
    """Codes and scales of rows, for caches to start from."""
    scale = x.float().abs().amax(-1) / MOST[codes]
    y = x.float() / torch.where(scale == 0, 1.0, scale)[..., None]
    return (y.round() if codes == torch.int8 else y).to(codes), scale


def norm(x, weight, eps):
    """x [.., dim] -> (normed, how far it may be off): sums of squares in 32 bits in any order of at most 16 + 5 additions
    after one another are off by 21 2^-24, their root by half of that, and the root's own error (2^-23) and the two products add
    four more: 2^-19 covers these 15 2^-24."""
    x = x.double().cpu()
    if weight is None:
        return x, torch.zeros_like(x)
    y = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * weight.double().cpu()
    return y, y.abs() * 2.0 ** -19


def stored_rows(want, off, codes, scale):
    """Whether codes [rows, dim] and scales [rows] are what rows `want`, known to `off`, are stored as."""
    want, off, scale = want.cpu(), off.cpu(), scale.double().cpu()
    c = codes.cpu().to(torch.float32).double()
    most = MOST[codes.dtype]
    top, slack = want.abs().amax(-1), off.amax(-1)
    # the greatest may be off by `slack`, and the division rounds
    assert bool(((scale - top / most).abs() <= slack / most + top / most * 2.0 ** -23).all())
    # half a step: of integers 1, of e4m3 2^-3 of the power of two below, 2^-9 at least; x / scale is off by a few 2^-24
    step = torch.ones_like(c)
    if codes.dtype != torch.int8:
        step = torch.exp2(torch.floor(torch.log2((want / scale.clamp(min=1e-300)[:, None]).abs().clamp(min=2.0 ** -6))) - 3)
    d = (c * scale[:, None] - want).abs()
    assert bool((d <= (0.5 * step + 2.0 ** -21 * most) * scale[:, None] + 2 * off + 1e-300).all()), float((d / scale[:, None]).max())


def poison(codes, scale, used, g):
    """Fills the rows that no position has: codes of any bits, scales that are not finite or huge."""
    junk = torch.randint(0, 256, codes.shape, generator=g, device=codes.device).to(torch.uint8).view(torch.int8)
    codes.view(torch.int8).copy_(torch.where(used[:, None, :, None], codes.view(torch.int8), junk))
    bad = torch.tensor([math.nan, math.inf, -math.inf, 3e38], device=scale.device)
    scale.copy_(torch.where(used[:, None, :], scale, bad[torch.randint(0, 4, scale.shape, generator=g, device=scale.device)]))


def attend(q, k, v, place, scale):
    """q [rows, dim] of one head, k and v [keys, dim] in 64 bits, place [rows] -> (out, how far it may be off).  As with a 16-bit
    cache: a score is a sum of dim products in 32 bits, and its key's scale; a probability takes the score's error twice, the
    exponential's, and with its value's scale one rounding to the type.  fp16 has fixed steps of 2^-24 there: a probability of
    1 is kept at 2^7 at least, and a scale in units of at most four times the greatest, so that half a step is 2^-25 2^-7 4
    = 2^-30 of the greatest value for each key."""
    u, dim = U[q.dtype], q.shape[1]
    if k.shape[0] == 0:
        z = torch.zeros_like(q, dtype=torch.float64)
        return z, z.clone()
    q = q.double()
    seen = torch.arange(k.shape[0], device=q.device) <= place[:, None]
    s = ((q @ k.T) * scale).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = p.sum(-1, keepdim=True)
    div = torch.where(total == 0, 1.0, total)
    o, size = p @ v / div, p @ v.abs() / div
    ds = (dim + 2) * 2.0 ** -24 * scale * ((q.abs() @ k.abs().T) * seen).amax(-1, keepdim=True)
    off = u * o.abs() + (u + 2 * ds + 2.0 ** -18) * size + 1e-7
    if u < 2.0 ** -8:
        off += 2.0 ** -30 * v.abs().max() * seen.sum(-1, keepdim=True) / div
    return o, off


def rows_of(c, cache, i, h, n, first=None, shared=0):
    """Keys and values [n, dim] of sequence i and head h, in 64 bits; the first `shared` positions from sequence `first`'s pages."""
    out = []
    for codes, scale in cache:
        at = torch.arange(n, device=codes.device)
        p = c.table[i, at // c.page].long()
        if shared:
            p = torch.where(at < shared, c.table[first, (at // c.page).clamp(max=c.table.shape[1] - 1)].long(), p)
        x = codes.view(torch.int8)[p, h, at % c.page].view(codes.dtype) if scale is not None else codes[p, h, at % c.page]
        out.append(x.double() if scale is None else values(x, scale[p, h, at % c.page]))
    return out


def attend_batch(c, q, cu):
    """All sequences and heads of a Case8: q [T, hq, dim] -> out, off (nan where no sequence has a row)."""
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    off = torch.zeros_like(out)
    for i, n in enumerate(c.kv_len):
        a, b = cu[i], cu[i + 1]
        if a == b:
            continue
        place = torch.arange(n - (b - a), n, device=q.device)
        for h in range(c.hkv):
            k, v = rows_of(c, ((c.kc, c.ks), (c.vc, c.vs)), i, h, n)
            for j in range(h * (c.hq // c.hkv), (h + 1) * (c.hq // c.hkv)):
                out[a:b, j], off[a:b, j] = attend(q[a:b, j], k, v, place, c.dim ** -0.5)
    return out, off


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rand(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Case8:
    """Sequences in an 8-bit cache of shuffled pages, with junk wherever no position is."""

    def __init__(self, hq, hkv, dim, page, dtype, codes, kv_len, seed=0, extra_cols=2, **desc):
        g = gen(seed)
        self.hq, self.hkv, self.dim, self.page, self.dtype, self.kv_len = hq, hkv, dim, page, dtype, kv_len
        per = [-(-n // page) for n in kv_len]
        total = sum(per) + 3
        order = torch.randperm(total, generator=g, device="cuda")[: sum(per)].to(torch.int32)
        # columns behind a sequence's pages name no page of the cache
        self.table = torch.full((len(kv_len), max(per + [1]) + extra_cols), 1 << 30, dtype=torch.int32, device="cuda")
        used = torch.zeros(total, page, dtype=torch.bool, device="cuda")
        at = 0
        for i, (n, p) in enumerate(zip(kv_len, per)):
            self.table[i, :p] = order[at: at + p]
            for c in range(p):
                used[order[at + c], : min(page, n - c * page)] = True
            at += p
        (self.kc, self.ks), (self.vc, self.vs) = (quantised(rand(g, total, hkv, page, dim), codes) for _ in range(2))
        poison(self.kc, self.ks, used, g)
        poison(self.vc, self.vs, used, g)
        self.att = qe_mixer.Attention(hq, hkv, dim, page, dtype=dtype, **desc)
        self.g = g

    def cache(self):
        return qe_mixer.Cache8(self.kc, self.vc, self.ks, self.vs)

    def copy(self):
        return qe_mixer.Cache8(self.kc.clone(), self.vc.clone(), self.ks.clone(), self.vs.clone())

    def batch(self, cu=None, **kw):
        return qe_mixer.Batch(ints(self.kv_len), self.table, None if cu is None else ints(cu), **kw)

    def q(self, T, std=2.0):
        return rand(self.g, T, self.hq, self.dim, dtype=self.dtype, std=std)


def bits(x):
    return x.view({1: torch.int8, 2: torch.int16, 4: torch.int32}[x.element_size()])


def same(a, b):
    """Whether two caches hold the same bits."""
    return all(torch.equal(bits(x), bits(y)) for x, y in ((a.kc, b.kc), (a.vc, b.vc), (a.k_scale, b.k_scale), (a.v_scale, b.v_scale)))
