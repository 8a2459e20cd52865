"""8-bit caches and norms from their definitions, in 64 bits, and the distances their kernels may be off."""
import math

import torch

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
