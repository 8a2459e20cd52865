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


def offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,dim,page", HEADS)
def test_prompt(hq, hkv, dim, page, dtype, codes):
    lens, ctx = [1, 0, 17, 200, 64, 5, 130], [0, 30, 40, 0, 64, 1000, 3]
    c = Case8(hq, hkv, dim, page, dtype, codes, [a + b for a, b in zip(lens, ctx)])
    cu = offsets(lens)
    q = c.q(cu[-1] + 3)  # rows behind the last sequence
    out = torch.full_like(q, 7.0)
    c.att.prompt8(c.batch(cu), q, c.cache(), out)
    c.att.check()
    want, off = Q.attend_batch(c, q[: cu[-1]], cu)
    close(out[: cu[-1]], want, off)
    assert bool((out[cu[-1]:] == 7).all())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("hq,hkv,dim,page,lens", [(16, 2, 256, 256, [1500, 600]), (32, 16, 256, 32, [900, 333]), (32, 8, 128, 64, [1500, 600]),
                                                  (24, 8, 64, 16, [1500, 600])])
def test_prompt_long(hq, hkv, dim, page, lens, codes):
    c = Case8(hq, hkv, dim, page, torch.bfloat16, codes, [lens[0], lens[1] + 300])
    cu = offsets(lens)
    q = c.q(cu[-1])
    out = torch.empty_like(q)
    c.att.prompt8(c.batch(cu), q, c.cache(), out)
    close(out, *Q.attend_batch(c, q, cu))


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dim,page", [(256, 256), (128, 16), (64, 64)])
def test_prompt_few_rows_over_a_long_cache(dim, page, codes):
    c = Case8(8, 2, dim, page, torch.float16, codes, [9000, 4097])
    cu = [0, 5, 6]
    q = c.q(6)
    want, off = Q.attend_batch(c, q, cu)
    for max_len in (0, 9000, 300):
        out = torch.empty_like(q)
        c.att.prompt8(c.batch(cu, max_len=max_len), q, c.cache(), out)
        close(out, want, off)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_rows_without_positions_are_zeros(dim):
    for extra in (2, 1000):  # one split, and several
        c = Case8(8, 2, dim, 16, torch.float16, torch.float8_e4m3fn, [3, 0, 20, 1500], extra_cols=extra)
        cu = [0, 10, 14, 34, 40]
        q = c.q(40)
        out = torch.full_like(q, 7.0)
        c.att.prompt8(c.batch(cu), q, c.cache(), out)
        c.att.check()
        close(out, *Q.attend_batch(c, q, cu))
        assert bool((out[:7] == 0).all()) and bool((out[10:14] == 0).all()) and bool((out[7] != 0).any())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("hq,hkv,dim,rows", [(8, 2, 64, 200), (8, 2, 128, 200), (16, 2, 256, 200), (32, 16, 256, 900)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_prompt_scales_that_are_not_finite_reach_their_rows_only(hq, hkv, dim, rows, which, codes):
    c = Case8(hq, hkv, dim, 16, torch.bfloat16, codes, [rows, 40])
    cu = [0, rows, rows + 40]
    q = c.q(cu[-1])
    want, off = Q.attend_batch(c, q, cu)
    for at in (0, 77, rows - 1):
        s = c.ks if which == "k" else c.vs
        place = int(c.table[0, at // 16]), 1, at % 16
        kept = s[place].clone()
        s[place] = math.nan if at else math.inf
        out = torch.empty_like(q)
        c.att.prompt8(c.batch(cu), q, c.cache(), out)
        group = hq // hkv
        gone = torch.zeros(cu[-1], hq, dtype=torch.bool, device="cuda")
        gone[at: rows, group: 2 * group] = True
        assert not bool(torch.isfinite(out[gone]).all(-1).any()) if which == "v" else bool(torch.isnan(out[gone][:, 0]).any())
        close(out[~gone], want[~gone], off[~gone])
        s[place] = kept


@pytest.mark.parametrize("codes", CODES)
def test_prompt_scales_of_any_size(codes):
    for dim in (64, 128, 256):
        c = Case8(8, 2, dim, 32, torch.float16, codes, [300, 200])
        cu = [0, 300, 310]
        q = c.q(310)
        c.ks *= torch.where(torch.arange(c.page, device="cuda") % 3 == 0, 2.0 ** -40, 1.0)
        c.vs *= torch.exp2(torch.arange(c.page, device="cuda") % 7 * 4.0 - 30.0)
        out = torch.empty_like(q)
        c.att.prompt8(c.batch(cu), q, c.cache(), out)
        close(out, *Q.attend_batch(c, q, cu))


@pytest.mark.parametrize("hq,hkv,dim,page,lens,extra_cols", [
    (8, 2, 128, 16, [500, 300, 20], 2), (4, 2, 64, 32, [300, 170, 33], 1500), (16, 4, 256, 64, [300, 40, 3], 2), (16, 1, 256, 16, [5, 9, 1], 2000),
    (32, 16, 256, 32, [1500, 600, 20], 2)])  # row blocks of four and of eight waves, one split and several
def test_bad_pages_give_zeros_for_all_rows_of_a_prompt(hq, hkv, dim, page, lens, extra_cols):
    ctx = [7, 1100, 0]
    c = Case8(hq, hkv, dim, page, torch.bfloat16, torch.int8, [a + b for a, b in zip(lens, ctx)], extra_cols=extra_cols)
    cu = offsets(lens)
    q = c.q(cu[-1])
    want, off = Q.attend_batch(c, q, cu)
    for i in range(2):
        pages = -(-c.kv_len[i] // page)
        for where, what in ((0, -1), (pages // 2, c.kc.shape[0]), (pages - 1, (1 << 31) - 1)):
            bad = c.table.clone()
            bad[i, where] = what
            out = torch.full_like(q, 7.0)
            c.att.prompt8(qe_mixer.Batch(ints(c.kv_len), bad, ints(cu)), q, c.cache(), out)
            with pytest.raises(qe_moe.QeError, match="page"):
                c.att.check()
            assert bool((out[cu[i]: cu[i + 1]] == 0).all()), (i, where)
            rest = torch.ones(cu[-1], dtype=torch.bool, device="cuda")
            rest[cu[i]: cu[i + 1]] = False
            close(out[rest], want[rest], off[rest])
    c.att.check()


@pytest.mark.parametrize("hq,hkv,dim,ctx,extra_cols", [(8, 2, 64, 0, 2), (16, 1, 256, 4000, 2), (4, 4, 128, 0, 2000)])  # one split, and several
def test_prompt_bad_lengths_and_offsets_give_zeros_and_an_error(hq, hkv, dim, ctx, extra_cols):
    lens = [170, 230, 100]
    c = Case8(hq, hkv, dim, 16, torch.bfloat16, torch.float8_e4m3fn, [n + ctx for n in lens], extra_cols=extra_cols)
    q = c.q(500)
    want, off = Q.attend_batch(c, q, [0, 170, 400, 500])
    for cu, kv1, lost in (([-5, 170, 400, 500], 0, [(0, 170)]), ([-7, -7, 400, 500], 0, [(0, 400)]), ([0, 170, 400, 501], 0, [(400, 500)]),
                          ([0, 170, 1 << 30, 1 << 30], 0, [(170, 500)]), ([0, 170, 400, 500], -1, [(170, 400)]), ([0, 170, 400, 500], 1 << 30, [(170, 400)])):
        out = torch.full_like(q, 7.0)
        kv = list(c.kv_len)
        kv[1] = kv1 or kv[1]
        c.att.prompt8(qe_mixer.Batch(ints(kv), c.table, ints(cu)), q, c.cache(), out)
        with pytest.raises(qe_moe.QeError, match="length or token offset"):
            c.att.check()
        gone = torch.zeros(500, dtype=torch.bool, device="cuda")
        for a, b in lost:
            gone[a:b] = True
        assert bool((out[gone] == 0).all()), cu
        if cu[1] == 170:
            close(out[~gone], want[~gone], off[~gone])


@pytest.mark.parametrize("n", [64, 65, 150])
@pytest.mark.parametrize("hq,hkv,dim,codes", [(8, 2, 128, torch.int8), (4, 4, 64, torch.float8_e4m3fn), (16, 1, 256, torch.int8)])
def test_prompt_of_many_sequences(hq, hkv, dim, codes, n):
    """Tiles are begun in the order of their sequences' lengths, among up to 64 sequences: equal ones, and ones without rows."""
    lens = [(7 * i) % 23 if i % 5 else 40 for i in range(n)]
    ctx = [(31 * i) % 400 if i % 3 else 100 - lens[i] for i in range(n)]
    c = Case8(hq, hkv, dim, 32, torch.bfloat16, codes, [a + b for a, b in zip(lens, ctx)])
    cu = offsets(lens)
    q = c.q(cu[-1])
    want, off = Q.attend_batch(c, q, cu)
    for max_len in (450, 20000):
        out = torch.full_like(q, 7.0)
        c.att.prompt8(c.batch(cu, max_len=max_len), q, c.cache(), out)
        c.att.check()
        close(out, want, off)


@pytest.mark.parametrize("hq,hkv,dim,lens,ctx", [(32, 8, 128, [300, 500], [40, 0]), (8, 2, 64, [20, 300], [5000, 0]), (16, 2, 256, [30, 7], [6000, 0])])
def test_prompt_and_decode_in_place(hq, hkv, dim, lens, ctx):
    c = Case8(hq, hkv, dim, 64, torch.bfloat16, torch.int8, [a + b for a, b in zip(lens, ctx)])
    cu = offsets(lens)
    q = c.q(cu[-1])
    out = torch.empty_like(q)
    c.att.prompt8(c.batch(cu), q, c.cache(), out)
    both = q.clone()
    c.att.prompt8(c.batch(cu), both, c.cache(), both)
    assert torch.equal(both, out)
    q = c.q(2)
    out = torch.empty_like(q)
    c.att.decode8(c.batch(), q, c.cache(), out)
    both = q.clone()
    c.att.decode8(c.batch(), both, c.cache(), both)
    assert torch.equal(both, out)
    c.att.check()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,dim", [(8, 2, 64), (32, 8, 128), (16, 1, 256)])
def test_a_row_of_one_key_is_its_value(hq, hkv, dim, dtype, codes):
    """But for the result's rounding.  Single tokens: a probability as two numbers of the type is off by U^2.  Prompts: its rounding is in the
    weights' sum, too, which has a few roundings of 2^-24 and a reciprocal's 2^-23."""
    n = 9
    c = Case8(hq, hkv, dim, 16, dtype, codes, [1] * n)
    q = c.q(n)
    want = torch.stack([torch.cat([Q.rows_of(c, ((c.vc, c.vs),), i, h, 1)[0] for h in range(hkv)]) for i in range(n)]).repeat_interleave(hq // hkv, 1)
    out = torch.empty_like(q)
    c.att.decode8(c.batch(), q, c.cache(), out)
    assert bool(((out.double() - want).abs() <= (Q.U[dtype] + 2 * Q.U[dtype] ** 2 + 2.0 ** -20) * want.abs() + 1e-7).all())
    c.att.prompt8(c.batch(list(range(n + 1))), q, c.cache(), out)
    assert bool(((out.double() - want).abs() <= (Q.U[dtype] + 2.0 ** -20) * want.abs() + 1e-7).all())
    # the first rows of prompts, beside rows of more keys
    c = Case8(hq, hkv, dim, 16, dtype, codes, [300, 70])
    q, out = c.q(370), torch.empty(370, hq, dim, dtype=dtype, device="cuda")
    c.att.prompt8(c.batch([0, 300, 370]), q, c.cache(), out)
    for i, row in ((0, 0), (1, 300)):
        want = torch.cat([Q.rows_of(c, ((c.vc, c.vs),), i, h, 1)[0] for h in range(hkv)]).repeat_interleave(hq // hkv, 0)
        assert bool(((out[row].double() - want).abs() <= (Q.U[dtype] + 2.0 ** -20) * want.abs() + 1e-7).all())


def in_halves(c, T, n_seqs, max_len):
    """Whether eight waves share a tile of such a call, as its plan has it."""
    tiles = (T * (c.hq // c.hkv) // 128 + n_seqs) * c.hkv
    return -(-max_len // 64) > 4 and 128 < tiles <= 256 or -(-max_len // 64) >= 16 and 256 < tiles <= 512


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,dim,page,lens,ctx", [
    (32, 8, 128, 16, [1, 33, 0, 700, 129], [0, 900, 5, 0, 63]), (32, 8, 128, 64, [1000, 200, 5], [24, 900, 1]),
    (12, 12, 64, 32, [1, 33, 0, 900, 513], [0, 1900, 5, 0, 64]), (24, 8, 64, 256, [300, 64, 65, 128, 40], [1000, 0, 0, 0, 3000]),
    (14, 2, 128, 16, [1, 1, 1, 1300], [0, 62, 63, 64])])
def test_prompt_in_halves(hq, hkv, dim, page, lens, ctx, dtype, codes):
    c = Case8(hq, hkv, dim, page, dtype, codes, [a + b for a, b in zip(lens, ctx)])
    cu = offsets(lens)
    q = c.q(cu[-1] + 3)
    want, off = Q.attend_batch(c, q[: cu[-1]], cu)
    for max_len in (3900, 1030):  # the host may have believed less
        assert in_halves(c, cu[-1] + 3, len(lens), max_len)
        out, again = torch.full_like(q, 7.0), torch.empty_like(q)
        c.att.prompt8(c.batch(cu, max_len=max_len), q, c.cache(), out)
        c.att.prompt8(c.batch(cu, max_len=max_len), q, c.cache(), again)
        c.att.check()
        close(out[: cu[-1]], want, off)
        assert bool((out[cu[-1]:] == 7).all()) and torch.equal(out[: cu[-1]], again[: cu[-1]])


@pytest.mark.parametrize("hq,hkv,dim", [(32, 8, 128), (24, 8, 64)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_prompt_in_halves_scales_that_are_not_finite(hq, hkv, dim, which):
    rows = 700
    c = Case8(hq, hkv, dim, 16, torch.float16, torch.int8, [rows, 40])
    cu = [0, rows, rows + 40]
    q = c.q(cu[-1])
    want, off = Q.attend_batch(c, q, cu)
    for at in (0, 77, rows - 1):  # of either half's steps
        s = c.ks if which == "k" else c.vs
        place = int(c.table[0, at // 16]), 1, at % 16
        kept = s[place].clone()
        s[place] = math.nan
        out = torch.empty_like(q)
        assert in_halves(c, cu[-1], 2, rows)
        c.att.prompt8(c.batch(cu, max_len=rows), q, c.cache(), out)
        gone = torch.zeros(cu[-1], hq, dtype=torch.bool, device="cuda")
        gone[at: rows, hq // hkv: 2 * (hq // hkv)] = True
        assert bool(torch.isnan(out[gone]).any(-1).all())
        close(out[~gone], want[~gone], off[~gone])
        s[place] = kept


@pytest.mark.parametrize("hq,hkv,dim", [(32, 8, 128), (24, 8, 64)])
def test_prompt_in_halves_bad_pages_lengths_and_scales_of_any_size(hq, hkv, dim):
    lens, ctx = [500, 300, 20, 30], [7, 1100, 0, -20]  # the last's first rows have no position
    c = Case8(hq, hkv, dim, 16, torch.float16, torch.int8, [a + b for a, b in zip(lens, ctx)])
    c.vs *= torch.exp2(torch.arange(c.page, device="cuda") % 7 * 4.0 - 30.0)
    cu = offsets(lens)
    q = c.q(cu[-1])
    assert in_halves(c, cu[-1], 4, 1400)
    want, off = Q.attend_batch(c, q, cu)
    out = torch.full_like(q, 7.0)
    c.att.prompt8(c.batch(cu, max_len=1400), q, c.cache(), out)
    c.att.check()
    close(out, want, off)
    assert bool((out[cu[3]: cu[3] + 20] == 0).all())
    for i, kv, where in ((0, None, 31), (1, None, 0), (1, -1, None), (0, 1 << 30, None)):
        bad, lengths = c.table.clone(), list(c.kv_len)
        if kv is None:
            bad[i, where] = c.kc.shape[0]
        else:
            lengths[i] = kv
        out = torch.full_like(q, 7.0)
        c.att.prompt8(qe_mixer.Batch(ints(lengths), bad, ints(cu), max_len=1400), q, c.cache(), out)
        with pytest.raises(qe_moe.QeError, match="page" if kv is None else "length"):
            c.att.check()
        rest = torch.ones(cu[-1], dtype=torch.bool, device="cuda")
        rest[cu[i]: cu[i + 1]] = False
        assert bool((out[~rest] == 0).all())
        close(out[rest], want[rest], off[rest])


@pytest.mark.parametrize("hq,hkv,dim,max_len", [(32, 8, 128, 2000), (24, 8, 64, 2000), (16, 2, 256, 0), (8, 2, 128, 2000)])  # halves, and splits
def test_prompts_captured_follow_lengths_and_offsets(hq, hkv, dim, max_len):
    """Rows of 900 tokens, shared out anew among three sequences before each replay: the order in which tiles are begun changes, too."""
    plans = [([300, 500, 100], [0, 0, 1500]), ([100, 0, 800], [1200, 300, 0]), ([1, 898, 1], [0, 900, 1990]), ([300, 500, 100], [0, 0, 1500])]
    most = [max(p[0][i] + p[1][i] for p in plans) for i in range(3)]
    c = Case8(hq, hkv, dim, 32, torch.float16, torch.int8, most)
    kv, cu = ints(most), ints([0, 300, 800, 900])
    batch = qe_mixer.Batch(kv, c.table, cu, max_len=max_len)
    q = c.q(900)
    out = torch.empty_like(q)
    c.att.prompt8(batch, q, c.cache(), out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.att.prompt8(batch, q, c.cache(), out, stream=torch.cuda.current_stream())
    for lens, ctx in plans:
        c.kv_len = [a + b for a, b in zip(lens, ctx)]
        kv.copy_(ints(c.kv_len))
        cu.copy_(ints(offsets(lens)))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        close(out, *Q.attend_batch(c, q, offsets(lens)))
        eager = torch.empty_like(out)
        c.att.prompt8(batch, q, c.cache(), eager)
        assert torch.equal(eager, out)
    c.att.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_of_zero_beside_great_ones(dtype):
    """A row of zeros has the scale 0, and its share of a row's weights."""
    for dim in (64, 128, 256):
        c = Case8(8, 2, dim, 16, dtype, torch.int8, [200, 7, 90])
        rows = torch.arange(c.page, device="cuda") % 3 == 0
        c.vs[:, :, rows] = 0
        c.vs[:, :, 1] *= 64
        q = c.q(60)
        out = torch.empty_like(q)
        c.att.prompt8(c.batch([0, 40, 44, 60]), q, c.cache(), out)
        close(out, *Q.attend_batch(c, q, [0, 40, 44, 60]))
        c.att.decode8(c.batch(), q[:3], c.cache(), out[:3])
        close(out[:3], *Q.attend_batch(c, q[:3], [0, 1, 2, 3]))
        c.att.check()


def test_far_offsets_in_a_large_cache():
    """Pages whose codes start past 2^32 bytes."""
    hkv, dim, page = 2, 256, 256
    pages = (1 << 32) // (hkv * page * dim) + 40
    c = Case8(16, hkv, dim, page, torch.bfloat16, torch.int8, [700, 513])
    kc, vc = (torch.empty(pages, hkv, page, dim, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(pages, hkv, page, device="cuda") for _ in range(2))
    far = ints([[pages - 1, 5, pages - 7], [3, pages - 2, 0]])
    for p, to in zip(c.table[:, :3].flatten().tolist(), far.flatten().tolist()):
        for a, b in ((kc, c.kc), (vc, c.vc), (ks, c.ks), (vs, c.vs)):
            a[to] = b[p]
    cache = qe_mixer.Cache8(kc, vc, ks, vs)
    q = c.q(90)
    want, off = Q.attend_batch(c, q[:2], [0, 1, 2])
    out = torch.empty_like(q)
    c.att.decode8(qe_mixer.Batch(ints(c.kv_len), far), q[:2], cache, out[:2])
    close(out[:2], want, off)
    c.att.prompt8(qe_mixer.Batch(ints(c.kv_len), far, ints([0, 60, 90])), q, cache, out)
    close(out, *Q.attend_batch(c, q, [0, 60, 90]))


def test_refusals():
    c = Case8(8, 2, 64, 32, torch.float16, torch.int8, [50, 60])
    q = c.q(2)
    out, a = torch.empty_like(q), c.att
    with pytest.raises(qe_moe.QeError, match="cu_q"):
        a.prompt8(c.batch(), q, c.cache(), out)
    with pytest.raises(qe_moe.QeError, match="cu_q"):
        a.decode8(c.batch([0, 1, 2]), q, c.cache(), out)
    other = Case8(8, 4, 64, 32, torch.float16, torch.int8, [50, 60])
    for call, b in ((a.prompt8, c.batch([0, 1, 2])), (a.decode8, c.batch())):
        for bad in (dict(q=q.float()), dict(q=q.cpu()), dict(q=q[:, :4]), dict(out=out.bfloat16()), dict(cache=other.cache())):
            with pytest.raises(ValueError):
                call(b, **{**dict(q=q, cache=c.cache(), out=out), **bad})
        cache = c.cache()
        cache.c.type = 1
        with pytest.raises(qe_moe.QeError, match="cache type"):
            call(b, q, cache, out)
        cache = c.cache()
        cache.c.k_scale = None
        with pytest.raises(qe_moe.QeError, match="scales"):
            call(b, q, cache, out)
        cache = c.cache()
        cache.c.v += 8
        with pytest.raises(qe_moe.QeError, match="aligned"):
            call(b, q, cache, out)
    a.check()
