"""The codes of an 8-bit cache are x / scale rounded to nearest, next to a border between two codes as well."""
import math

import pytest

torch = pytest.importorskip("torch")
import cache8_ref as Q  # noqa: E402
from cache8_ref import Case8, gen  # noqa: E402

pytestmark = pytest.mark.gpu


def border_rows(codes, rows, dim, seed):
    """Float32 rows, each with a greatest element of any size and the others next to where two codes meet: the product of the border
    and the row's scale in 32 bits, and its neighbours on either side."""
    g = torch.Generator().manual_seed(seed)
    most = Q.MOST[codes]
    top = torch.exp2(torch.rand(rows, 1, generator=g) * 200 - 95)
    scale = top / most
    if codes == torch.int8:
        border = torch.randint(0, 127, (rows, dim), generator=g).float() + 0.5
    else:  # of the 16 steps of a power of two the odd 32nds, and of the smallest ones the odd multiples of 2^-10
        power = torch.exp2(torch.randint(-6, 9, (rows, dim), generator=g).float())
        border = power * (1 + (2 * torch.randint(0, 8, (rows, dim), generator=g).float() + 1) / 16)
        small = (2 * torch.randint(0, 8, (rows, dim), generator=g).float() + 1) * 2.0 ** -10
        border = torch.where(torch.rand(rows, dim, generator=g) < 0.25, small, border).clamp(max=most)
    x = border * scale
    step = torch.randint(-1, 2, (rows, dim), generator=g)
    x = torch.where(step < 0, torch.nextafter(x, torch.zeros(())), torch.where(step > 0, torch.nextafter(x, torch.full((), math.inf)), x))
    x = torch.minimum(x, top) * torch.where(torch.rand(rows, dim, generator=g) < 0.5, -1.0, 1.0)
    x[torch.arange(rows), torch.randint(0, dim, (rows,), generator=g)] = top[:, 0]
    return x


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("hkv,dim", [(2, 256), (8, 128), (3, 64)])
def test_codes_next_to_borders(hkv, dim, codes):
    n = 500
    x = border_rows(codes, n * hkv, dim, 3 * dim + hkv)
    scale = x.abs().amax(-1) / Q.MOST[codes]
    y = x / scale[:, None]
    want = (y.round() if codes == torch.int8 else y).to(codes)
    c = Case8(hkv, hkv, dim, 32, torch.bfloat16, codes, [n])
    cache, rows = c.copy(), x.view(n, hkv, dim).cuda()
    c.att.append8(c.batch([0, n]), None, rows, rows, cache, None)
    c.att.check()
    at = torch.arange(n, device="cuda")
    p, r = c.table[0, at // 32].long(), at % 32
    for cc, s in ((cache.kc, cache.k_scale), (cache.vc, cache.v_scale)):  # (no rotation: k is as it is, too)
        assert torch.equal(s[p, :, r].reshape(-1).cpu(), scale)
        got = cc.view(torch.int8)[p, :, r].reshape(-1, dim).cpu()
        wrong = got != want.view(torch.int8)
        assert not bool(wrong.any()), (int(wrong.sum()), wrong.numel())


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_codes_of_16_bit_rows(codes):
    """Elements of few bits are often halves of a step: all of them are bfloat16 numbers."""
    g = gen(1)
    n, dim = 700, 128
    x = (torch.randint(-255, 256, (n, 1, dim), generator=g, device="cuda").float() / 2).bfloat16()
    x[:, 0, 0] = 127.0
    c = Case8(1, 1, dim, 16, torch.bfloat16, codes, [n])
    cache = c.copy()
    c.att.append8(c.batch([0, n]), None, x, x, cache, None)
    c.att.check()
    y = x[:, 0].float().cpu()
    scale = y.abs().amax(-1) / Q.MOST[codes]
    z = y / scale[:, None]
    want = (z.round() if codes == torch.int8 else z).to(codes).view(torch.int8)
    at = torch.arange(n, device="cuda")
    got = cache.kc.view(torch.int8)[c.table[0, at // 16].long(), 0, at % 16].cpu()
    assert torch.equal(got, want)
