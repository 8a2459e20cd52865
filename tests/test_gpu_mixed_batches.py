"""Calls of random geometries over 8-bit caches: ragged batches with empty sequences, rows before the first position, scales of several sizes,
groups of none to nine, hints that are exact, absent or wrong."""
import math
import random

import pytest

torch = pytest.importorskip("torch")
import cache8_ref as Q  # noqa: E402
from cache8_ref import Case8  # noqa: E402
from test_gpu_shared import Grouped  # noqa: E402

pytestmark = pytest.mark.gpu


def close(out, want, off):
    assert torch.isfinite(out).all()
    d = (out.double() - want).abs()
    assert bool((d <= off).all()), float((d / off.clamp(min=1e-30)).max())


def more(off, want, dtype):
    """cache8_ref.attend's bound, for one rounding e_i of each weight w_i, is u sum w |v| beside the result's own.  Where the rounded weights are summed (prompts'
    rows of few keys, shared positions) the result is off by the sum of e_i w_i (v_i - o), which is u (sum w |v| + |o|) at most."""
    return off + Q.U[dtype] * want.abs()


@pytest.mark.parametrize("seed", range(24))
def test_random_calls(seed):
    rng = random.Random(seed)

    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    group, hkv, dim, page = rng.randint(1, 16), rng.randint(1, 6), rng.choice((64, 128, 256)), rng.choice((16, 32, 64, 128, 256))
    dtype, codes = rng.choice((torch.bfloat16, torch.float16)), rng.choice((torch.int8, torch.float8_e4m3fn))
    n = spread(1, 30)
    lens = [rng.choice((0, 1, 1, spread(1, 300))) for _ in range(n)]
    kv = [max(0, x + rng.choice((0, spread(1, 3000), -rng.randint(0, 5)))) for x in lens]
    c = Case8(group * hkv, hkv, dim, page, dtype, codes, kv, extra_cols=rng.choice((1, 3, 700)), seed=seed)
    if rng.random() < 0.4:
        c.vs *= torch.exp2(torch.arange(page, device="cuda") % 5 * 3.0 - 12.0)
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    hints = (0, max(max(kv), 1), rng.randint(1, 4000))
    if cu[-1]:
        q = c.q(cu[-1])
        want, off = Q.attend_batch(c, q, cu)
        for h in hints:
            out = torch.full_like(q, 7.0)
            c.att.prompt8(c.batch(cu, max_len=h), q, c.cache(), out)
            c.att.check()
            close(out, want, more(off, want, dtype))
    q = c.q(n)
    want, off = Q.attend_batch(c, q, list(range(n + 1)))
    for h in hints:
        out = torch.full_like(q, 7.0)
        c.att.decode8(c.batch(max_len=h), q, c.cache(), out)
        c.att.check()
        close(out, want, off)
    members = [rng.randint(0, 9) for _ in range(rng.randint(1, 4))] + [1]
    prefix = [rng.choice((0, spread(1, 4000))) if m else 0 for m in members]
    before, behind = rng.randint(0, 2), rng.randint(0, 2)
    own = [rng.choice((0, 1, spread(1, 2500))) for _ in range(sum(members) + before + behind)]
    cache = rng.choice((None, codes))
    g = Grouped((group * hkv, hkv, dim, page), dtype, cache, members, own, prefix, before=before, behind=behind, seed=seed)
    q = g.c.q(len(own))
    want, off = g.expect(q)
    off = off if cache is None else more(off, want, dtype)
    for h in ((0, 0), (max(max(g.c.kv_len), 1), max(prefix)), (rng.randint(1, 5000), rng.randint(1, 5000))):
        out = torch.full_like(q, 7.0)
        g.run(q, out, *h)
        g.c.att.check()
        close(out, want, off)
