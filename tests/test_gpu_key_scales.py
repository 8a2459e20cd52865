"""A key's scale that is NaN makes NaN of every row that attends to its position, and one that is infinite of no other row."""
import math

import pytest

torch = pytest.importorskip("torch")
import cache8_ref as Q  # noqa: E402
from cache8_ref import Case8, ints  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("dtype,codes", [(torch.bfloat16, torch.int8), (torch.float16, torch.float8_e4m3fn), (torch.float16, torch.int8)])
@pytest.mark.parametrize("hq,hkv,dim,rows,ctx,max_len", [(8, 2, 64, 200, 0, 0), (8, 2, 128, 150, 70, 0), (16, 2, 256, 100, 30, 150), (32, 16, 256, 900, 0, 900),
                                                         (32, 8, 128, 700, 0, 740), (8, 1, 256, 9, 3000, 0)])  # rows of eight waves, halves, splits
def test_prompt(hq, hkv, dim, rows, ctx, max_len, dtype, codes, which):
    c = Case8(hq, hkv, dim, 16, dtype, codes, [rows + ctx, 40])
    cu = [0, rows, rows + 40]
    q = c.q(cu[-1])
    want, off = Q.attend_batch(c, q, cu)
    s, group = c.ks if which == "k" else c.vs, hq // hkv
    for at in (0, 7, ctx, ctx + rows // 2, ctx + rows - 1):
        place = int(c.table[0, at // 16]), hkv - 1, at % 16
        kept = s[place].clone()
        gone = torch.zeros(cu[-1], hq, dtype=torch.bool, device="cuda")
        gone[max(at - ctx, 0): rows, hq - group:] = True
        for bad in (math.nan, math.inf, -math.inf):
            s[place] = bad
            out = torch.full_like(q, 7.0)
            c.att.prompt8(c.batch(cu, max_len=max_len), q, c.cache(), out)
            c.att.check()
            if bad != bad:
                assert bool(torch.isnan(out[gone]).all()), at
            assert torch.isfinite(out[~gone]).all()
            assert bool(((out[~gone].double() - want[~gone]).abs() <= off[~gone]).all()), (at, bad)
        s[place] = kept


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("dtype,codes", [(torch.bfloat16, torch.int8), (torch.float16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_single_tokens(dim, dtype, codes, which):
    import qe_mixer

    c = Case8(8, 2, dim, 16, dtype, codes, [900, 40, 33])
    q = c.q(3)
    want, off = Q.attend_batch(c, q, [0, 1, 2, 3])
    s = c.ks if which == "k" else c.vs
    for at in (0, 500, 899):
        place = int(c.table[0, at // 16]), 1, at % 16
        kept = s[place].clone()
        s[place] = math.nan
        for groups in (None, ([0, 1], [600]), ([0, 0, 1], [5, 0])):
            out = torch.full_like(q, 7.0)
            if groups is None:
                c.att.decode8(c.batch(), q, c.cache(), out)
            else:
                c.att.decode8_shared(c.batch(), qe_mixer.Shared(ints(groups[0]), ints(groups[1])), q, c.cache(), out)
            c.att.check()
            assert bool(torch.isnan(out[0, 4:]).all()), (at, groups)
            assert bool(((out[0, :4].double() - want[0, :4]).abs() <= off[0, :4]).all())
            assert bool(((out[1:].double() - want[1:]).abs() <= off[1:]).all())
        s[place] = kept
