"""Values behind a row's causal limit, however much greater than its own, leave the row as exact as it is without them."""
import math

import pytest

torch = pytest.importorskip("torch")
import cache8_ref as Q  # noqa: E402
from cache8_ref import Case8  # noqa: E402

pytestmark = pytest.mark.gpu


def offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


@pytest.mark.parametrize("ratio", [22, 32, 90])
@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,dim,lens,ctx,max_len", [
    (8, 2, 64, [200, 30], [0, 0], 0), (8, 2, 128, [200, 30], [0, 500], 600), (16, 2, 256, [120, 200], [0, 40], 300), (3, 3, 128, [100, 64], [0, 0], 200),
    (32, 16, 256, [900, 333], [0, 30], 1000),  # eight waves of rows
    (32, 8, 128, [300, 200, 333], [0, 60, 0], 400),  # eight waves in halves
    (16, 1, 256, [7, 40], [3000, 2000], 0)])  # several splits
def test_prompt(hq, hkv, dim, lens, ctx, max_len, dtype, codes, ratio):
    """Positions at, and right behind, the borders of a wave's rows, of a tile and of a page have values 2^ratio times as great as the others.
    The bound is that of rows that have only the positions before the first of them (cache8_ref.attend: the greatest value is theirs)."""
    c = Case8(hq, hkv, dim, 16, dtype, codes, [a + b for a, b in zip(lens, ctx)])
    c.vs *= 2.0 ** -8
    cu = offsets(lens)
    q = c.q(cu[-1])
    kept = c.vs.clone()
    for back in (1, 2, 6, 31, 40, 65):  # from the last position
        c.vs.copy_(kept)
        at = []
        for i, n in enumerate(c.kv_len):
            at.append(max(n - back, ctx[i] + 1))
            p, r = c.table[i, at[i] // 16].long(), at[i] % 16
            c.vs[p, :, r:] *= 2.0 ** ratio
            for x in range(at[i] // 16 + 1, -(-n // 16)):
                c.vs[c.table[i, x].long()] *= 2.0 ** ratio
        out = torch.full_like(q, 7.0)
        c.att.prompt8(c.batch(cu, max_len=max_len), q, c.cache(), out)
        c.att.check()
        for i in range(len(lens)):
            n = at[i] - ctx[i]  # rows before
            place = torch.arange(ctx[i], at[i], device="cuda")
            for h in range(hkv):
                k, v = Q.rows_of(c, ((c.kc, c.ks), (c.vc, c.vs)), i, h, at[i])
                for j in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    got = out[cu[i]: cu[i] + n, j]
                    want, off = Q.attend(q[cu[i]: cu[i] + n, j], k, v, place, dim ** -0.5)
                    assert torch.isfinite(got).all(), (back, i, j)
                    d = (got.double() - want).abs()
                    assert bool((d <= off).all()), (back, i, j, float((d / off).max()))


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_prompts_first_row_is_its_value_beside_later_great_ones(dim, codes):
    """As test_a_row_of_one_key_is_its_value has it, where the second position's values are 2^20 times as great."""
    c = Case8(8, 2, dim, 16, torch.float16, codes, [90])
    c.vs *= 2.0 ** -8
    c.vs[c.table[0, 0].long(), :, 1:] *= 2.0 ** 20
    q, out = c.q(90), torch.empty(90, 8, dim, dtype=torch.float16, device="cuda")
    c.att.prompt8(c.batch([0, 90]), q, c.cache(), out)
    want = torch.cat([Q.rows_of(c, ((c.vc, c.vs),), 0, h, 1)[0] for h in range(2)]).repeat_interleave(4, 0)
    u = Q.U[torch.float16]
    # half a step of a result below fp16's normal range, 2^-25, beside what a row of one key may be off by
    assert bool(((out[0].double() - want).abs() <= (u + 2.0 ** -20) * want.abs() + 2.0 ** -25).all())
    assert math.isfinite(float(out[0].float().sum()))
