"""Attention over an 8-bit cache against its definition in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
import cache8_ref as Q  # noqa: E402
import qe_mixer  # noqa: E402
import qe_moe  # noqa: E402
from cache8_ref import Case8, ints, rand  # noqa: E402

pytestmark = pytest.mark.gpu
HEADS = [(16, 2, 256, 256), (32, 8, 128, 64), (14, 2, 128, 32), (3, 3, 64, 16), (16, 1, 64, 128), (1, 1, 256, 16)]
CODES = [torch.int8, torch.float8_e4m3fn]


def close(out, want, off):
    assert torch.isfinite(out).all()
    d = (out.double() - want).abs()
    assert bool((d <= off).all()), float((d / off).max())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,dim,page", HEADS)
def test_decode(hq, hkv, dim, page, dtype, codes):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 0]
    c = Case8(hq, hkv, dim, page, dtype, codes, lens)
    q = c.q(len(lens))
    out = torch.full_like(q, 7.0)
    c.att.decode8(c.batch(), q, c.cache(), out)
    c.att.check()
    close(out, *Q.attend_batch(c, q, list(range(len(lens) + 1))))
    assert bool((out[-1] == 0).all())  # a sequence without positions


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("hq,hkv,dim,page", [(16, 2, 256, 256), (8, 8, 64, 16), (14, 2, 128, 32)])
@pytest.mark.parametrize("n", [129, 5000, 40000])
def test_decode_split_over_a_long_sequence(hq, hkv, dim, page, n, codes):
    c = Case8(hq, hkv, dim, page, torch.bfloat16, codes, [n, 7])
    q = c.q(2)
    want, off = Q.attend_batch(c, q, [0, 1, 2])
    for max_len in (0, n, 1):  # the hint changes the split, not the result
        out = torch.empty_like(q)
        c.att.decode8(c.batch(max_len=max_len), q, c.cache(), out)
        close(out, want, off)


def test_decode_many_sequences():
    n = 300
    lens = [1 + 37 * i % 211 for i in range(n)]
    c = Case8(8, 8, 64, 32, torch.float16, torch.int8, lens)
    q = c.q(n)
    out = torch.empty_like(q)
    c.att.decode8(c.batch(), q, c.cache(), out)
    close(out, *Q.attend_batch(c, q, list(range(n + 1))))
    c.att.check()


def test_decode_rows_with_strides_and_in_place():
    c = Case8(16, 2, 256, 64, torch.bfloat16, torch.int8, [300, 20, 77])
    wide = rand(c.g, 3, 20, 256, dtype=torch.bfloat16)
    q = wide[:, :16]
    want, off = Q.attend_batch(c, q.contiguous(), [0, 1, 2, 3])
    outs = torch.full((3, 18 * 256), 5.0, dtype=torch.bfloat16, device="cuda")
    c.att.decode8(c.batch(), q, c.cache(), outs[:, : 16 * 256])
    close(outs[:, : 16 * 256].reshape(3, 16, 256), want, off)
    assert bool((outs[:, 16 * 256:] == 5).all())
    c.att.decode8(c.batch(), q, c.cache(), q)
    close(q, want, off)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode_scales_of_any_size(dtype, codes):
    """Values far beyond and below fp16's range in their codes' scales; keys whose scales differ by 2^40."""
    c = Case8(8, 2, 128, 32, dtype, codes, [100, 700])
    q = c.q(2)
    c.ks *= torch.where(torch.arange(c.page, device="cuda") % 3 == 0, 2.0 ** -40, 1.0)
    c.vs *= torch.exp2(torch.arange(c.page, device="cuda") % 7 * 4.0 - 30.0)
    out = torch.empty_like(q)
    c.att.decode8(c.batch(), q, c.cache(), out)
    close(out, *Q.attend_batch(c, q, [0, 1, 2]))
    if dtype == torch.bfloat16:
        c.vs *= 2.0 ** 80
        c.att.decode8(c.batch(), q, c.cache(), out)
        close(out, *Q.attend_batch(c, q, [0, 1, 2]))


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("n", [20, 3000])
def test_decode_rows_that_are_not_finite_reach_their_sequence_only(n, which):
    c = Case8(8, 2, 128, 32, torch.bfloat16, torch.int8, [n, 50])
    q = c.q(2)
    want, off = Q.attend_batch(c, q, [0, 1, 2])
    (c.ks if which == "k" else c.vs)[int(c.table[0, 0]), 1, 5] = math.nan
    out = torch.empty_like(q)
    c.att.decode8(c.batch(), q, c.cache(), out)
    assert bool(torch.isnan(out[0, 4:]).all())
    close(out[0, :4], want[0, :4], off[0, :4])
    close(out[1], want[1], off[1])


@pytest.mark.parametrize("n", [40, 3000])
def test_decode_bad_pages_and_lengths_give_zeros_and_an_error(n):
    c = Case8(8, 2, 64, 32, torch.float16, torch.float8_e4m3fn, [n, 60])
    q = c.q(2)
    want, off = Q.attend_batch(c, q, [0, 1, 2])
    good = c.table.clone()
    for at in (0, (n - 1) // 32):
        for wrong in (-1, c.kc.shape[0], (1 << 31) - 1):
            c.table.copy_(good)
            c.table[0, at] = wrong
            out = torch.full_like(q, 7.0)
            c.att.decode8(c.batch(), q, c.cache(), out)
            with pytest.raises(qe_moe.QeError, match="page"):
                c.att.check()
            assert bool((out[0] == 0).all())
            close(out[1], want[1], off[1])
    c.table.copy_(good)
    for wrong in (-1, c.table.shape[1] * 32 + 1, (1 << 31) - 1, -(1 << 31)):
        b = qe_mixer.Batch(ints([n, wrong]), c.table)
        out = torch.full_like(q, 7.0)
        c.att.decode8(b, q, c.cache(), out)
        with pytest.raises(qe_moe.QeError, match="length"):
            c.att.check()
        assert bool((out[1] == 0).all())
        close(out[0], want[0], off[0])
