"""Attention over the paged cache, and the rotary cache write, against their definitions in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
import mixer_ref as R  # noqa: E402
import qe_mixer  # noqa: E402
import qe_moe  # noqa: E402

pytestmark = pytest.mark.gpu
HEADS = [(16, 2, 256, 256), (32, 8, 128, 64), (14, 2, 128, 32), (3, 3, 64, 16), (16, 1, 64, 128), (1, 1, 256, 16)]


def rand(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Case:
    """Sequences in a cache of shuffled pages, with NaN and infinities wherever no position is."""

    def __init__(self, hq, hkv, dim, page, dtype, kv_len, seed=0, extra_cols=2, **desc):
        g = gen(seed)
        self.hq, self.hkv, self.dim, self.page, self.dtype, self.kv_len = hq, hkv, dim, page, dtype, kv_len
        per = [-(-n // page) for n in kv_len]
        total = sum(per) + 3
        self.kc, self.vc = (rand(g, total, hkv, page, dim, dtype=dtype) for _ in range(2))
        order = torch.randperm(total, generator=g, device="cuda")[: sum(per)].to(torch.int32)
        # columns behind a sequence's pages name no page of the cache
        self.table = torch.full((len(kv_len), max(per + [1]) + extra_cols), 1 << 30, dtype=torch.int32, device="cuda")
        poison = torch.tensor([math.nan, math.inf, -math.inf, 3e38 if dtype == torch.bfloat16 else 6e4], device="cuda", dtype=dtype)
        free = torch.ones(total, page, dtype=torch.bool, device="cuda")
        at = 0
        for i, (n, p) in enumerate(zip(kv_len, per)):
            self.table[i, :p] = order[at: at + p]
            for c in range(p):
                free[order[at + c], : min(page, n - c * page)] = False
            at += p
        for c in (self.kc, self.vc):
            fill = poison[torch.randint(0, 4, c.shape, generator=g, device="cuda")]
            c.copy_(torch.where(free[:, None, :, None], fill, c))
        self.att = qe_mixer.Attention(hq, hkv, dim, page, dtype=dtype, **desc)
        self.g = g

    def batch(self, cu=None, **kw):
        return qe_mixer.Batch(ints(self.kv_len), self.table, None if cu is None else ints(cu), **kw)

    def q(self, T, std=2.0):
        return rand(self.g, T, self.hq, self.dim, dtype=self.dtype, std=std)

    def expect(self, q, cu):
        return R.attend_batch(q, self.kc, self.vc, self.table, self.kv_len, cu, self.dim ** -0.5, self.page)


def close(out, want, off):
    d = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    assert bool((d <= off).all()), float((d / off).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,dim,page", HEADS)
def test_decode(hq, hkv, dim, page, dtype):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 0]
    c = Case(hq, hkv, dim, page, dtype, lens)
    q = c.q(len(lens))
    out = torch.full_like(q, 7.0)
    c.att.decode(c.batch(), q, c.kc, c.vc, out)
    c.att.check()
    close(out, *c.expect(q, list(range(len(lens) + 1))))
    assert bool((out[-1] == 0).all())  # a sequence without positions


@pytest.mark.parametrize("hq,hkv,dim,page", [(16, 2, 256, 256), (8, 8, 64, 16), (14, 2, 128, 32)])
@pytest.mark.parametrize("n", [129, 5000, 33333])
def test_decode_split_over_a_long_sequence(hq, hkv, dim, page, n):
    c = Case(hq, hkv, dim, page, torch.bfloat16, [n, 7])
    q = c.q(2)
    want, off = c.expect(q, [0, 1, 2])
    for max_len in (0, n, 1):  # the hint changes the split, not the result
        out = torch.empty_like(q)
        c.att.decode(c.batch(max_len=max_len), q, c.kc, c.vc, out)
        close(out, want, off)


def test_many_sequences():
    """More sequences times heads than a decode call has workgroups for splits, in all three calls."""
    n, page = 300, 32
    lens = [1 + 37 * i % 211 for i in range(n)]
    c = Case(8, 8, 64, page, torch.float16, lens)
    k, v = rand(c.g, n, 8, 64, dtype=torch.float16), rand(c.g, n, 8, 64, dtype=torch.float16)
    for b in (c.batch(), c.batch(list(range(n + 1)))):
        kc, vc = c.kc.clone(), c.vc.clone()
        c.att.append(b, None, k, v, kc, vc, None)
        c.att.check()
        for i, at in enumerate(lens):
            p, row = int(c.table[i, (at - 1) // page]), (at - 1) % page
            assert torch.equal(kc[p, :, row], k[i]) and torch.equal(vc[p, :, row], v[i]), i
    q = c.q(n)
    want, off = c.expect(q, list(range(n + 1)))
    for attend, b in ((c.att.decode, c.batch()), (c.att.prompt, c.batch(list(range(n + 1))))):
        out = torch.empty_like(q)
        attend(b, q, c.kc, c.vc, out)
        close(out, want, off)
    c.att.check()


def test_calls_without_tokens():
    c = Case(4, 2, 64, 16, torch.bfloat16, [0, 20], rotary=64)
    kc, vc = c.kc.clone(), c.vc.clone()
    q, k = c.q(0), rand(c.g, 0, 2, 64, dtype=torch.bfloat16)
    c.att.append(c.batch([0, 0, 0]), q, k, k, c.kc, c.vc, torch.empty_like(q))
    c.att.prompt(c.batch([0, 0, 0]), q, c.kc, c.vc, torch.empty_like(q))
    q, k, out = c.q(3), rand(c.g, 3, 2, 64, dtype=torch.bfloat16), torch.full((3, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    c.att.append(c.batch([3, 3, 3]), q, k, k, c.kc, c.vc, out)  # rows, but of no sequence
    c.att.prompt(c.batch([0, 0, 0]), q, c.kc, c.vc, out)
    c.att.check()
    assert bool((out == 7).all())
    assert torch.equal(kc.view(torch.int16), c.kc.view(torch.int16)) and torch.equal(vc.view(torch.int16), c.vc.view(torch.int16))


def test_decode_rows_with_strides_and_in_place():
    c = Case(16, 2, 256, 64, torch.bfloat16, [300, 20, 77])
    wide = rand(c.g, 3, 20, 256, dtype=torch.bfloat16)
    q = wide[:, :16]
    want, off = c.expect(q.contiguous(), [0, 1, 2, 3])
    outs = torch.full((3, 18 * 256), 5.0, dtype=torch.bfloat16, device="cuda")
    c.att.decode(c.batch(), q, c.kc, c.vc, outs[:, : 16 * 256])
    close(outs[:, : 16 * 256].reshape(3, 16, 256), want, off)
    assert bool((outs[:, 16 * 256:] == 5).all())
    rest = wide[:, 16:].clone()
    c.att.decode(c.batch(), q, c.kc, c.vc, q)
    close(q, want, off)
    assert torch.equal(wide[:, 16:], rest)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,dim,page", HEADS)
def test_prompt(hq, hkv, dim, page, dtype):
    lens = [1, 0, 17, 200, 64, 5, 130]
    ctx = [0, 30, 40, 0, 64, 1000, 3]
    c = Case(hq, hkv, dim, page, dtype, [a + b for a, b in zip(lens, ctx)])
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    q = c.q(cu[-1] + 3)  # rows behind the last sequence
    out = torch.full_like(q, 7.0)
    c.att.prompt(c.batch(cu), q, c.kc, c.vc, out)
    c.att.check()
    want, off = c.expect(q[: cu[-1]], cu)
    close(out[: cu[-1]], want, off)
    assert bool((out[cu[-1]:] == 7).all())


@pytest.mark.parametrize("hq,hkv,dim,page", [(16, 2, 256, 256), (32, 8, 128, 64), (24, 8, 64, 16)])
def test_prompt_long(hq, hkv, dim, page):
    c = Case(hq, hkv, dim, page, torch.bfloat16, [1500, 900])
    cu = [0, 1500, 2100]
    q = c.q(2100)
    out = torch.empty_like(q)
    c.att.prompt(c.batch(cu), q, c.kc, c.vc, out)
    close(out, *c.expect(q, cu))


@pytest.mark.parametrize("dim,page", [(256, 256), (128, 16), (64, 64)])
def test_prompt_few_rows_over_a_long_cache(dim, page):
    c = Case(8, 2, dim, page, torch.float16, [9000, 4097])
    cu = [0, 5, 6]
    q = c.q(6)
    want, off = c.expect(q, cu)
    for max_len in (0, 9000, 300):
        out = torch.empty_like(q)
        c.att.prompt(c.batch(cu, max_len=max_len), q, c.kc, c.vc, out)
        close(out, want, off)


@pytest.mark.parametrize("hq,hkv,dim", [(32, 8, 128), (16, 4, 256), (24, 8, 64)])
def test_prompt_many_rows_over_many_splits(hq, hkv, dim):
    c = Case(hq, hkv, dim, 32, torch.bfloat16, [2600, 2700])
    cu = [0, 100, 260]
    q = c.q(260)
    out = torch.empty_like(q)
    c.att.prompt(c.batch(cu, max_len=2700), q, c.kc, c.vc, out)
    c.att.check()
    close(out, *c.expect(q, cu))


@pytest.mark.parametrize("hq,hkv,dim,lens,kv", [(32, 8, 128, (60, 70), (2600, 2700)), (24, 8, 64, (60, 110), (2700, 2500)), (16, 2, 256, (150, 151), (2560, 3000))])
def test_prompt_more_than_eight_splits_of_more_than_4096_rows(hq, hkv, dim, lens, kv):
    """One wave joins a row's splits there, however many they are."""
    c = Case(hq, hkv, dim, 64, torch.float16, list(kv))
    cu = [0, lens[0], sum(lens)]
    tiles = (cu[2] * (hq // hkv) // 128 + 2) * hkv
    assert tiles * 128 > 4096 and min(512 // tiles, -(-max(kv) // 256)) > 8  # the plan's, with row blocks of 128
    q = c.q(cu[2])
    out = torch.empty_like(q)
    c.att.prompt(c.batch(cu, max_len=max(kv)), q, c.kc, c.vc, out)
    c.att.check()
    close(out, *c.expect(q, cu))


@pytest.mark.parametrize("dim,n,below", [(64, 1 << 20, 26.0), (128, 100000, 25.1), (256, 40000, 27.0), (64, 3000, 20.0)])
@pytest.mark.parametrize("first", [True, False])  # the great one's place
def test_fp16_keys_far_below_the_greatest_count(dim, n, below, first):
    """One key's score is above all others', whose weights fp16 does not hold at their own size, but together they are
    0.03 to 1.5 % of the row's."""
    page, scale = 256, dim ** -0.5
    pages = -(-n // page)
    kc, vc = (torch.zeros(pages, 1, page, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.arange(pages, device="cuda", dtype=torch.int32)[None]
    at = 0 if first else n - 1
    kc[at // page, 0, at % page, 3] = 1.0
    vc[:, 0] = torch.linspace(0.5, 2.0, dim, device="cuda").half()
    vc[at // page, 0, at % page] = 0
    q = torch.zeros(1, 2, dim, dtype=torch.float16, device="cuda")
    q[:, 0, 3], q[:, 1, 3] = below * math.log(2) / scale, (below - 3) * math.log(2) / scale
    att = qe_mixer.Attention(2, 1, dim, page, dtype=torch.float16)
    for h in range(2):
        want, _ = R.attend(q[:, h], kc.view(-1, dim)[:n], vc.view(-1, dim)[:n], torch.tensor([n - 1], device="cuda"), scale)
        score = float(q[0, h, 3]) * scale
        # as for all rows: a rounding of the result and one of the probabilities, the score's in 32 bits, the exponential's; and
        # half of the fixed steps of fp16, 2^-25, at 2^15 and (prompts) at least 2^7 times the size, for each key
        near = want.abs() * (2 * 2.0 ** -11 + 2 * dim * 2.0 ** -24 * score + 2.0 ** -18)
        for up, cu in ((15, None), (7, ints([0, 1]))):
            out = torch.empty_like(q)
            (att.decode if cu is None else att.prompt)(qe_mixer.Batch(ints([n]), table, cu), q, kc, vc, out)
            off = near + n * 2.0 ** (-25 - up) * 2.0
            assert bool(((out[:, h].double() - want).abs() <= off).all()), (h, up, float(((out[:, h].double() - want).abs() / want).max()))
    att.check()


def test_prompt_rows_without_positions_are_zeros():
    c = Case(8, 2, 128, 16, torch.bfloat16, [3, 0, 20])
    cu = [0, 10, 14, 34]  # ten tokens of which three are in the cache, four of which none is
    q = c.q(34)
    out = torch.full_like(q, 7.0)
    c.att.prompt(c.batch(cu), q, c.kc, c.vc, out)
    want, off = c.expect(q, cu)
    close(out, want, off)
    assert bool((out[:7] == 0).all()) and bool((out[10:14] == 0).all()) and bool((out[7] != 0).any())


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_rows_without_positions_are_zeros_in_several_splits(dim):
    c = Case(8, 2, dim, 16, torch.float16, [3, 0, 20, 1500], extra_cols=1000)
    cu = [0, 10, 14, 34, 40]
    q = c.q(40)
    out = torch.full_like(q, 7.0)
    c.att.prompt(c.batch(cu), q, c.kc, c.vc, out)
    c.att.check()
    close(out, *c.expect(q, cu))
    assert bool((out[:7] == 0).all()) and bool((out[10:14] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_values_that_are_not_finite_reach_their_rows_only(dim, dtype):
    n = 150
    c = Case(4, 2, dim, 32, dtype, [n])
    q = c.q(n)
    clean = torch.empty_like(q)
    c.att.prompt(c.batch([0, n]), q, c.kc, c.vc, clean)
    for at, what in ((70, math.nan), (131, math.inf), (149, -math.inf)):
        k, v = c.kc.clone(), c.vc.clone()
        p, row = int(c.table[0, at // 32]), at % 32
        v[p, 0, row, dim - 3] = what
        out = torch.empty_like(q)
        c.att.prompt(c.batch([0, n]), q, c.kc, v, out)
        assert torch.equal(out[:at], clean[:at])
        assert torch.equal(out[:, 2:], clean[:, 2:])  # the other key-value head's
        hit = out[at:, :2, dim - 3]
        assert bool((hit.isnan() if what != what else hit == what).all())
        keep = [d for d in range(dim) if d != dim - 3]
        assert torch.equal(out[at:, :2, keep], clean[at:, :2, keep])
        k[p, 1, row] = math.nan
        c.att.prompt(c.batch([0, n]), q, k, c.vc, out)
        assert torch.equal(out[:at], clean[:at]) and torch.equal(out[:, :2], clean[:, :2]) and bool(out[at:, 2:].isnan().all())


def test_prompt_of_many_rows_and_heads_of_256():
    """Enough row blocks of 256 for every CU: workgroups of eight waves."""
    c = Case(32, 16, 256, 32, torch.bfloat16, [1600, 700, 33])
    cu = [0, 1500, 2100, 2101]
    q = c.q(2110)
    clean = torch.full_like(q, 7.0)
    c.att.prompt(c.batch(cu), q, c.kc, c.vc, clean)
    c.att.check()
    close(clean[:2101], *c.expect(q[:2101], cu))
    assert bool((clean[2101:] == 7).all())
    v = c.vc.clone()
    for i, at, what in ((0, 1333, math.inf), (1, 699, math.nan)):  # positions: of a token in the middle, and of a last one
        v[int(c.table[i, at // 32]), 3, at % 32, 200] = what
    out = torch.full_like(q, 7.0)
    c.att.prompt(c.batch(cu), q, c.kc, v, out)
    hit = torch.zeros_like(q, dtype=torch.bool)
    hit[1333 - 100: 1500, 6:8, 200] = hit[2099, 6:8, 200] = True  # rows from those positions on, of the two heads that read them
    assert torch.equal(out[~hit], clean[~hit])
    assert bool((out[:1500][hit[:1500]] == math.inf).all()) and bool(out[1500:][hit[1500:]].isnan().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("extra_cols", [2, 700])  # one split; and one tile of keys each, so that some begin at their rows' own keys
def test_prompt_values_that_are_not_finite_in_a_workgroups_first_tile(dim, dtype, extra_cols):
    n = 150
    c = Case(4, 2, dim, 32, dtype, [n], extra_cols=extra_cols)
    q = c.q(n)
    clean, out = torch.empty_like(q), torch.empty_like(q)
    c.att.prompt(c.batch([0, n]), q, c.kc, c.vc, clean)
    for at, what in ((0, math.nan), (1, math.inf), (15, -math.inf), (16, math.nan), (31, math.inf), (32, math.nan), (47, math.inf), (48, math.nan),
                     (63, math.inf), (64, math.nan), (100, -math.inf), (128, math.nan), (148, math.inf)):
        v = c.vc.clone()
        v[int(c.table[0, at // 32]), 1, at % 32, dim - 1] = what
        c.att.prompt(c.batch([0, n]), q, c.kc, v, out)
        hit = torch.zeros_like(q, dtype=torch.bool)
        hit[at:, 2:, dim - 1] = True
        assert torch.equal(out[~hit], clean[~hit]), at
        assert bool((out[hit].isnan() if what != what else out[hit] == what).all()), at
    c.att.check()


def test_prompt_values_that_are_not_finite_in_the_first_tile_of_eight_waves():
    c = Case(32, 16, 256, 32, torch.bfloat16, [1500, 600])
    cu = [0, 1500, 2100]
    q = c.q(2100)
    clean, out = torch.empty_like(q), torch.empty_like(q)
    c.att.prompt(c.batch(cu), q, c.kc, c.vc, clean)
    for at, what in ((0, math.nan), (7, math.inf), (8, -math.inf), (31, math.nan), (32, math.inf), (55, math.nan), (63, math.inf)):
        v = c.vc.clone()
        for i in range(2):
            v[int(c.table[i, at // 32]), 5, at % 32, 129] = what
        c.att.prompt(c.batch(cu), q, c.kc, v, out)
        hit = torch.zeros_like(q, dtype=torch.bool)
        hit[at:1500, 10:12, 129] = hit[1500 + at:, 10:12, 129] = True
        assert torch.equal(out[~hit], clean[~hit]), at
        assert bool((out[hit].isnan() if what != what else out[hit] == what).all()), at
    c.att.check()


def test_far_offsets_in_a_large_cache():
    """Pages that start past 2^31 elements and 2^32 bytes."""
    hkv, dim, page = 2, 256, 256
    pages = (1 << 32) // (hkv * page * dim) + 40
    kc, vc = (torch.empty(pages, hkv, page, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = gen(3)
    table = ints([[pages - 1, 5, pages - 7], [3, pages - 2, 0]])
    for p in table.flatten().tolist():
        kc[p], vc[p] = rand(g, hkv, page, dim, dtype=torch.bfloat16), rand(g, hkv, page, dim, dtype=torch.bfloat16)
    att = qe_mixer.Attention(16, hkv, dim, page)
    kv = [700, 513]
    q = rand(g, 2, 16, dim, dtype=torch.bfloat16, std=2.0)
    out = torch.empty_like(q)
    att.decode(qe_mixer.Batch(ints(kv), table), q, kc, vc, out)
    close(out, *R.attend_batch(q, kc, vc, table, kv, [0, 1, 2], dim ** -0.5, page))
    q = rand(g, 90, 16, dim, dtype=torch.bfloat16, std=2.0)
    out = torch.empty_like(q)
    att.prompt(qe_mixer.Batch(ints(kv), table, ints([0, 60, 90])), q, kc, vc, out)
    close(out, *R.attend_batch(q, kc, vc, table, kv, [0, 60, 90], dim ** -0.5, page))
    k = rand(g, 2, hkv, dim, dtype=torch.bfloat16)
    att.append(qe_mixer.Batch(ints(kv), table), None, k, k, kc, vc, None)
    assert torch.equal(vc[pages - 7, :, 699 - 512], k[0]) and torch.equal(kc[0, :, 0], k[1])


# -- rotary positions and the cache write -----------------------------------------
@pytest.mark.parametrize("in_dtype", [torch.float32, None])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,dim,page,rotary,sections,interleaved", [
    (16, 2, 256, 256, 64, (11, 11, 10), True), (4, 2, 128, 16, 128, (64,), False), (3, 3, 64, 32, 48, (10, 8, 6), False),
    (2, 1, 64, 16, 64, (14, 9, 9), True), (2, 2, 64, 16, 0, (0,), False)])
def test_append(hq, hkv, dim, page, rotary, sections, interleaved, dtype, in_dtype):
    lens, ctx = [1, 40, 0, 3], [0, 100, 7, 261900]
    kv = [a + b for a, b in zip(lens, ctx)]
    kv[3] = 64  # a late position in an early row: positions are given, not counted
    c = Case(hq, hkv, dim, page, dtype, kv, rotary=rotary, theta=1e7, sections=sections, interleaved=interleaved)
    in_dtype = in_dtype or dtype
    T = sum(lens)
    qkv = rand(c.g, T + 2, hq + 2 * hkv, dim, dtype=in_dtype)
    q, k, v = qkv.split((hq, hkv, hkv), 1)
    axes = len(sections)
    pos = torch.randint(0, 262144, (axes, T + 2), generator=c.g, device="cuda").to(torch.int32)
    cu = [0, 1, 41, 41, 44]
    out = torch.full((T + 2, hq, dim), 7.0, dtype=dtype, device="cuda")
    kc, vc = c.kc.clone(), c.vc.clone()
    c.att.append(c.batch(cu), q, k, v, kc, vc, out, pos=pos)
    c.att.check()
    u = R.U[dtype]
    wq, oq = R.rotate(q, pos, rotary, 1e7, R.axes_of(rotary, sections, interleaved))
    wk, ok = R.rotate(k, pos, rotary, 1e7, R.axes_of(rotary, sections, interleaved))
    assert bool(((out[:T].double().cpu() - wq[:T]).abs() <= oq[:T] + u * wq[:T].abs() + 1e-7).all())
    assert bool((out[T:] == 7).all())
    used = torch.zeros(kc.shape[0], page, dtype=torch.bool)
    for i, n in enumerate(lens):
        for j in range(n):
            at, t = kv[i] - n + j, cu[i] + j
            p, row = int(c.table[i, at // page]), at % page
            used[p, row] = True
            d = (kc[p, :, row].double().cpu() - wk[t]).abs()
            assert bool((d <= ok[t] + u * wk[t].abs() + 1e-7).all()), (i, j)
            assert torch.equal(vc[p, :, row], v[t].to(dtype))
    rest = ~used[:, None, :, None].expand(kc.shape).cuda()
    for a, b in ((kc, c.kc), (vc, c.vc)):  # nothing else was written
        assert torch.equal(a.view(torch.int16)[rest], b.view(torch.int16)[rest])


def test_append_counts_positions_and_rotates_in_place():
    c = Case(4, 2, 64, 16, torch.float16, [35], rotary=64, theta=1e4)
    q, k, v = rand(c.g, 5, 4, 64, dtype=torch.float16), rand(c.g, 5, 2, 64, dtype=torch.float16), rand(c.g, 5, 2, 64, dtype=torch.float16)
    given, counted = torch.empty_like(q), q.clone()
    k2, v2 = c.kc.clone(), c.vc.clone()
    c.att.append(c.batch([0, 5]), q, k, v, c.kc, c.vc, given, pos=ints([[30, 31, 32, 33, 34]]))
    c.att.append(c.batch([0, 5]), counted, k, v, k2, v2, counted)
    assert torch.equal(given, counted) and torch.equal(c.kc.view(torch.int16), k2.view(torch.int16))
    assert not torch.equal(given, q)


def test_append_before_the_first_position_writes_nothing():
    c = Case(4, 2, 64, 16, torch.float16, [2], rotary=64)
    q, k = rand(c.g, 5, 4, 64, dtype=torch.float16), rand(c.g, 5, 2, 64, dtype=torch.float16)
    out, kc, vc = torch.empty_like(q), c.kc.clone(), c.vc.clone()
    c.att.append(c.batch([0, 5]), q, k, k, kc, vc, out, pos=ints([[0, 0, 0, 1, 2]]))
    c.att.check()
    p = int(c.table[0, 0])
    assert torch.equal(out[:3], q[:3])  # position 0 turns nothing
    assert torch.equal(vc[p, :, 0], k[3]) and torch.equal(vc[p, :, 1], k[4])
    vc[p, :, :2] = c.vc[p, :, :2]
    assert torch.equal(vc.view(torch.int16), c.vc.view(torch.int16))


# -- what device memory may hold ----------------------------------------------------
@pytest.mark.parametrize("n", [40, 3000])
def test_bad_pages_give_zeros_and_an_error(n):
    c = Case(8, 2, 128, 16, torch.bfloat16, [n, n])
    good = c.q(2)
    want, off = c.expect(good, [0, 1, 2])
    for where, page in ((0, -1), (1, c.kc.shape[0]), (n // 16 - 1, (1 << 31) - 1)):
        bad = c.table.clone()
        bad[0, where] = page
        for prompt in (False, True):
            b = qe_mixer.Batch(ints([n, n]), bad, ints([0, 1, 2]) if prompt else None)
            out = torch.full_like(good, 7.0)
            (c.att.prompt if prompt else c.att.decode)(b, good, c.kc, c.vc, out)
            with pytest.raises(qe_moe.QeError, match="page"):
                c.att.check()
            assert bool((out[0] == 0).all())
            close(out[1], want[1], off[1])
            c.att.check()  # reported once
    k = rand(c.g, 2, 2, 128, dtype=torch.bfloat16)
    kc, vc = c.kc.clone(), c.vc.clone()
    bad = c.table.clone()
    bad[0, (n - 1) // 16] = 1 << 30
    c.att.append(qe_mixer.Batch(ints([n, n]), bad), None, k, k, kc, vc, None)
    torch.cuda.synchronize()
    with pytest.raises(qe_moe.QeError, match="page") as e:  # the next call reports it too, and does nothing else
        c.att.append(c.batch(), None, k, k, kc, vc, None)
    assert e.value.code == qe_moe.QE_ERR_STATE
    p = int(c.table[1, (n - 1) // 16])
    assert torch.equal(kc[p, :, (n - 1) % 16], k[1])
    kc[p], vc[p] = c.kc[p], c.vc[p]
    assert torch.equal(kc.view(torch.int16), c.kc.view(torch.int16)) and torch.equal(vc.view(torch.int16), c.vc.view(torch.int16))


@pytest.mark.parametrize("hq,hkv,dim,page,lens,extra_cols", [
    (8, 2, 128, 16, [500, 300, 20], 2), (4, 2, 64, 32, [300, 170, 33], 1500), (16, 4, 256, 64, [300, 40, 3], 2), (16, 1, 256, 16, [5, 9, 1], 2000),
    (32, 16, 256, 32, [1500, 600, 20], 2)])  # row blocks of four and of eight waves, one split and several
def test_bad_pages_give_zeros_for_all_rows_of_a_prompt(hq, hkv, dim, page, lens, extra_cols):
    ctx = [7, 1100, 0]
    c = Case(hq, hkv, dim, page, torch.bfloat16, [a + b for a, b in zip(lens, ctx)], extra_cols=extra_cols)
    cu = [0, lens[0], lens[0] + lens[1], sum(lens)]
    q = c.q(cu[-1])
    want, off = c.expect(q, cu)
    for i in range(2):
        pages = -(-c.kv_len[i] // page)
        for where, what in ((0, -1), (pages // 2, c.kc.shape[0]), (pages - 1, (1 << 31) - 1)):
            bad = c.table.clone()
            bad[i, where] = what
            out = torch.full_like(q, 7.0)
            c.att.prompt(qe_mixer.Batch(ints(c.kv_len), bad, ints(cu)), q, c.kc, c.vc, out)
            with pytest.raises(qe_moe.QeError, match="page"):
                c.att.check()
            assert bool((out[cu[i]: cu[i + 1]] == 0).all()), (i, where)
            rest = torch.ones(cu[-1], dtype=torch.bool, device="cuda")
            rest[cu[i]: cu[i + 1]] = False
            close(out[rest], want[rest], off[rest])
    c.att.check()


@pytest.mark.parametrize("hq,hkv,dim,rows", [(2, 1, 64, 3), (16, 16, 256, 4000)])  # workgroups of 256 and of 512 threads
def test_bad_pages_anywhere_in_a_long_table_are_found(hq, hkv, dim, rows):
    page, n = 16, 5000 * 16 - 5
    kc, vc = (torch.ones(3, hkv, page, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.randint(0, 3, (1, 5001), generator=gen(1), device="cuda").to(torch.int32)
    table[0, 5000] = -1  # behind the sequence
    att = qe_mixer.Attention(hq, hkv, dim, page)
    q = rand(gen(2), rows, hq, dim, dtype=torch.bfloat16)
    out = torch.empty_like(q)
    for at in (None, 0, 1, 255, 256, 511, 512, 767, 768, 1023, 1024, 2047, 2048, 3333, 4095, 4096, 4999):
        bad = table.clone()
        if at is not None:
            bad[0, at] = 3 if at % 2 else -1
        att.prompt(qe_mixer.Batch(ints([n]), bad, ints([0, rows]), max_len=n), q, kc, vc, out)
        if at is None:
            att.check()
            assert bool(((out.float() - 1).abs() <= 2 * 2.0 ** -8).all())  # an average of ones
        else:
            with pytest.raises(qe_moe.QeError, match="page"):
                att.check()
            assert bool((out == 0).all()), at


def test_bad_lengths_give_zeros_and_an_error():
    c = Case(8, 2, 64, 32, torch.float16, [50, 60])
    q = c.q(2)
    want, off = c.expect(q, [0, 1, 2])
    for wrong in (-1, c.table.shape[1] * 32 + 1, (1 << 31) - 1, -(1 << 31)):
        for prompt in (False, True):
            b = qe_mixer.Batch(ints([wrong, 60]), c.table, ints([0, 1, 2]) if prompt else None)
            out = torch.full_like(q, 7.0)
            (c.att.prompt if prompt else c.att.decode)(b, q, c.kc, c.vc, out)
            with pytest.raises(qe_moe.QeError, match="length"):
                c.att.check()
            assert bool((out[0] == 0).all())
            close(out[1], want[1], off[1])
    b = qe_mixer.Batch(ints([50, 60]), c.table, ints([0, 1, 999]))
    c.att.prompt(b, q, c.kc, c.vc, torch.empty_like(q))
    with pytest.raises(qe_moe.QeError, match="offset"):
        c.att.check()


@pytest.mark.parametrize("cu", [[0, 1000, 500, 1000], [0, 1000, 0, 1000], [300, 200, 1000, 1000], [0, 10, 20, 10], [0, 1 << 30, 500, 1000]])
def test_offsets_that_fall_are_reported(cu):
    """Also where a sequence that they leave without rows is the only one to show it."""
    c = Case(1, 1, 64, 16, torch.bfloat16, [1000, 1000, 1000], rotary=64)
    q, k = c.q(1000), rand(c.g, 1000, 1, 64, dtype=torch.bfloat16)
    out, rot, kc, vc = torch.empty_like(q), torch.full_like(q, 7.0), c.kc.clone(), c.vc.clone()
    c.att.prompt(c.batch(cu), q, c.kc, c.vc, out)
    with pytest.raises(qe_moe.QeError, match="offset"):
        c.att.check()
    c.att.append(c.batch(cu), q, k, k, kc, vc, rot)
    with pytest.raises(qe_moe.QeError, match="offset"):
        c.att.check()
    # tokens of a sequence beside the fall are left out
    for i in range(3):
        if 0 <= cu[i] <= cu[i + 1] <= 1000 and (i == 0 or cu[i - 1] <= cu[i]) and (i == 2 or cu[i + 1] <= cu[i + 2]):
            continue
        p = c.table[i, : 1000 // 16].long()
        assert torch.equal(kc[p].view(torch.int16), c.kc[p].view(torch.int16)) and torch.equal(vc[p].view(torch.int16), c.vc[p].view(torch.int16))
    if cu[1] == 1000:  # here that is every token
        assert bool((rot == 7).all())


@pytest.mark.parametrize("hq,hkv,dim,ctx,extra_cols", [(8, 2, 64, 0, 2), (16, 1, 256, 4000, 2), (4, 4, 128, 0, 2000)])  # one split, and several
def test_offsets_outside_the_call_give_zeros_and_an_error(hq, hkv, dim, ctx, extra_cols):
    lens = [170, 230, 100]
    c = Case(hq, hkv, dim, 16, torch.bfloat16, [n + ctx for n in lens], extra_cols=extra_cols)
    q = c.q(500)
    want, off = c.expect(q, [0, 170, 400, 500])
    for cu, lost in (([-5, 170, 400, 500], [(0, 170)]), ([-100000, 170, 400, 500], [(0, 170)]), ([-7, -7, 400, 500], [(0, 400)]),
                     ([0, 170, 400, 501], [(400, 500)]), ([0, 170, 1 << 30, 1 << 30], [(170, 500)]), ([-(1 << 31), 170, 400, (1 << 31) - 1], [(0, 170), (400, 500)])):
        out = torch.full_like(q, 7.0)
        c.att.prompt(c.batch(cu), q, c.kc, c.vc, out)
        with pytest.raises(qe_moe.QeError, match="offset"):
            c.att.check()
        gone = torch.zeros(500, dtype=torch.bool, device="cuda")
        for a, b in lost:
            gone[a:b] = True
        assert bool((out[gone] == 0).all()), cu
        if cu[1] == 170:
            close(out[~gone], want[~gone], off[~gone])


def test_offsets_of_sequences_without_tokens_are_looked_at():
    n = 700
    c = Case(1, 1, 64, 16, torch.float16, [20, 3] + [0] * (n - 2), rotary=64)
    q, k = c.q(2), rand(c.g, 2, 1, 64, dtype=torch.float16)
    want, off = R.attend_batch(q, c.kc, c.vc, c.table, [20, 3], [0, 1, 2], 64 ** -0.5, 16)
    for at, what, word in ((None, 0, None), (n, 3, "offset"), (n - 1, 5, "offset"), (n - 100, 1, "offset"), (400, -1, "offset")):
        cu = [0, 1] + [2] * (n - 1)
        if at is not None:
            cu[at] = what
        b = c.batch(cu)
        out, rot, kc, vc = torch.empty_like(q), torch.empty_like(q), c.kc.clone(), c.vc.clone()
        for call in (lambda: c.att.append(b, q, k, k, kc, vc, rot), lambda: c.att.prompt(b, q, c.kc, c.vc, out)):
            call()
            if word:
                with pytest.raises(qe_moe.QeError, match=word):
                    c.att.check()
            else:
                c.att.check()
        if not word:
            close(out, want, off)
            assert torch.equal(vc[int(c.table[0, 1]), :, 3], k[0]) and torch.equal(vc[int(c.table[1, 0]), :, 2], k[1])


def test_refusals():
    c = Case(8, 2, 64, 32, torch.float16, [50, 60])
    q, k = c.q(2), rand(c.g, 2, 2, 64, dtype=torch.float16)
    out, a = torch.empty_like(q), c.att
    with pytest.raises(qe_moe.QeError):
        a.prompt(c.batch(), q, c.kc, c.vc, out)
    with pytest.raises(qe_moe.QeError):
        a.decode(c.batch([0, 1, 2]), q, c.kc, c.vc, out)
    with pytest.raises(qe_moe.QeError, match="n_tokens"):
        a.decode(c.batch(), c.q(3), c.kc, c.vc, c.q(3))
    for bad in (dict(q=q.float()), dict(q=q.cpu()), dict(q=q[:, :4]), dict(out=out.bfloat16()), dict(kc=c.kc.float()), dict(vc=c.vc[1:]),
                dict(kc=c.kc.transpose(1, 2)), dict(q=q.transpose(0, 1).contiguous().transpose(0, 1))):
        with pytest.raises(ValueError):
            a.decode(c.batch(), **{**dict(q=q, kc=c.kc, vc=c.vc, out=out), **bad})
    pad = torch.empty(2, 8 * 64 + 4, dtype=torch.float16, device="cuda")
    with pytest.raises(qe_moe.QeError, match="stride"):
        a.decode(c.batch(), pad[:, : 8 * 64], c.kc, c.vc, out)
    with pytest.raises(qe_moe.QeError, match="aligned"):
        a.decode(c.batch(), torch.empty(1025, dtype=torch.float16, device="cuda")[1:].view(2, 8, 64), c.kc, c.vc, out)
    with pytest.raises(ValueError):
        a.append(c.batch(), q, k, k, c.kc, c.vc, None)
    with pytest.raises(ValueError):
        a.append(c.batch(), q, k, k.float(), c.kc, c.vc, out)
    with pytest.raises(ValueError):
        a.append(c.batch(), q, k, k, c.kc, c.vc, out, pos=ints([[0]]))
    with pytest.raises(ValueError):
        qe_mixer.Batch(ints([1, 2]), c.table.long())
    with pytest.raises(ValueError):
        qe_mixer.Batch(ints([1, 2]).long(), c.table)
    with pytest.raises(ValueError):
        qe_mixer.Batch(ints([1, 2]), c.table, ints([0, 1]))
    b = c.batch()
    b.c.max_pages = b.c.table_stride = (1 << 30) // 32 + 1
    with pytest.raises(qe_moe.QeError, match="max_pages"):
        a.decode(b, q, c.kc, c.vc, out)
    many = qe_mixer.Attention(256, 256, 64, 16)
    n = 65535
    b = qe_mixer.Batch(torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, 1, dtype=torch.int32, device="cuda"),
                       torch.zeros(n + 1, dtype=torch.int32, device="cuda"))
    pages = torch.zeros(1, 256, 16, 64, dtype=torch.bfloat16, device="cuda")
    rows = torch.full((256, 256, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(qe_moe.QeError, match="threads"):
        many.prompt(b, rows, pages, pages, rows)
    many.check()
    a.check()


def test_tables_of_far_rows_are_refused():
    """Rows 2^32 + 8 apart are not rows 8 apart."""
    far = torch.empty((1 << 32) + 16, dtype=torch.int32, device="cuda")
    for kw in (dict(table=far.as_strided((2, 8), ((1 << 32) + 8, 1))), dict(table=far[:8].view(2, 4), max_len=(1 << 32) + 4)):
        with pytest.raises(ValueError, match="32 bits"):
            qe_mixer.Batch(ints([3, 4]), **kw)


# -- streams, graphs ------------------------------------------------------------------
def test_captured_calls_follow_the_lengths_in_device_memory():
    """append, prompt and decode in a graph, replayed as the sequences grow, with eager work between the replays."""
    c = Case(8, 2, 128, 16, torch.bfloat16, [600, 300], rotary=64, theta=1e6)
    g = c.g
    c.kc.copy_(rand(g, *c.kc.shape, dtype=torch.bfloat16)), c.vc.copy_(rand(g, *c.vc.shape, dtype=torch.bfloat16))
    kv = ints([200, 10])
    one = qe_mixer.Batch(kv, c.table)
    two = qe_mixer.Batch(kv, c.table, ints([0, 1, 2]))
    q, k, v = c.q(2), rand(g, 2, 2, 128, dtype=torch.bfloat16), rand(g, 2, 2, 128, dtype=torch.bfloat16)
    r, o1, o2 = (torch.empty_like(q) for _ in range(3))
    kc, vc = c.kc.clone(), c.vc.clone()

    def calls(stream, r, o1, o2, kc, vc):
        c.att.append(one, q, k, v, kc, vc, r, stream=stream)
        c.att.decode(one, r, kc, vc, o1, stream=stream)
        c.att.prompt(two, r, kc, vc, o2, stream=stream)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        calls(side, r, o1, o2, kc, vc)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(torch.cuda.current_stream(), r, o1, o2, kc, vc)
    for step in range(5):
        kv.copy_(ints([200 + 97 * step, 10 + 70 * step]))
        q.copy_(c.q(2)), k.copy_(rand(g, 2, 2, 128, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        e = [torch.empty_like(q) for _ in range(3)]
        calls(None, *e, c.kc, c.vc)
        torch.cuda.synchronize()
        for a, b in zip((r, o1, o2, kc, vc), (*e, c.kc, c.vc)):
            assert torch.equal(a, b), step
        off = R.attend_batch(r, c.kc, c.vc, c.table, kv.tolist(), [0, 1, 2], 128 ** -0.5, 16)
        close(o1, *off)
        close(o2, *off)


def test_two_graphs_share_a_context():
    """One after the other, and calls of other sizes between them: what a call leaves in the scratch is of no use to the next."""
    c = Case(16, 2, 256, 256, torch.bfloat16, [9000, 300, 2000])
    d = [(c.batch(), c.q(3)), (qe_mixer.Batch(ints([9000]), c.table[:1]), c.q(1)), (c.batch([0, 4, 5, 40]), c.q(40))]
    outs = [torch.empty_like(q) for _, q in d]
    want = [c.expect(d[0][1], [0, 1, 2, 3]), R.attend_batch(d[1][1], c.kc, c.vc, c.table, [9000], [0, 1], 1 / 16, 256),
            c.expect(d[2][1], [0, 4, 5, 40])]

    def call(i, stream=None):
        (c.att.prompt if i == 2 else c.att.decode)(*d[i], c.kc, c.vc, outs[i], stream=stream)

    graphs = []
    for i in (0, 1):
        call(i)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(i, torch.cuda.current_stream())
    for _ in range(4):
        for o in outs:
            o.fill_(7.0)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        call(2)
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            close(o, *w)
    c.att.check()


def test_contexts_on_streams_of_their_own():
    """Calls of two contexts that overlap share nothing: splits joined by the last workgroup, by a launch, and prompts'."""
    cs = [Case(16, 2, 256, 64, torch.bfloat16, [3000, 900], seed=s) for s in (1, 2)]
    qs, rows, streams = [c.q(2) for c in cs], [c.q(9) for c in cs], [torch.cuda.Stream() for _ in cs]
    long_ = [Case(16, 2, 256, 64, torch.bfloat16, [20000], seed=s) for s in (3, 4)]
    outs = [[(torch.empty_like(q), torch.empty_like(q[:1]), torch.empty_like(r)) for _ in range(6)] for q, r in zip(qs, rows)]
    bs = [(c.batch(), l.batch(), c.batch([0, 4, 9])) for c, l in zip(cs, long_)]
    torch.cuda.synchronize()
    for k in range(6):
        for i, s in enumerate(streams):
            a, b, p = outs[i][k]
            cs[i].att.decode(bs[i][0], qs[i], cs[i].kc, cs[i].vc, a, stream=s)
            long_[i].att.decode(bs[i][1], qs[i][:1], long_[i].kc, long_[i].vc, b, stream=s)
            cs[i].att.prompt(bs[i][2], rows[i], cs[i].kc, cs[i].vc, p, stream=s)
    for i, s in enumerate(streams):
        cs[i].att.check(s), long_[i].att.check(s)
        want = cs[i].expect(qs[i], [0, 1, 2]), long_[i].expect(qs[i][:1], [0, 1]), cs[i].expect(rows[i], [0, 4, 9])
        for got in outs[i]:
            for x, w in zip(got, want):
                close(x, *w)


def test_results_do_not_change_from_call_to_call():
    c = Case(16, 2, 256, 256, torch.bfloat16, [5000, 100])
    q, outs = c.q(2), [torch.empty(2, 16, 256, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    for o in outs:
        c.att.decode(c.batch(), q, c.kc, c.vc, o)
    assert all(torch.equal(o, outs[0]) for o in outs[1:])
