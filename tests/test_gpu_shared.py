"""Attention of single tokens whose sequences share their beginnings, against its definition in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
import cache8_ref as Q  # noqa: E402
import mixer_ref as R  # noqa: E402
import qe_mixer  # noqa: E402
import qe_moe  # noqa: E402
from cache8_ref import Case8, ints  # noqa: E402
from test_gpu_attention import Case  # noqa: E402

pytestmark = pytest.mark.gpu
CACHES = [None, torch.int8, torch.float8_e4m3fn]  # None: 16 bits
HEADS = [(16, 2, 256, 256), (32, 8, 128, 64), (14, 2, 128, 32), (3, 3, 64, 16), (16, 1, 64, 128), (1, 1, 256, 16)]


class Grouped:
    """A case whose groups' first sequences alone hold the shared positions: the others' tables name no page there, and the
    rows before them in the page where their own begin hold junk."""

    def __init__(self, heads, dtype, cache, groups, own, prefix, before=0, behind=0, seed=0):
        """groups: members of each; own: positions of each sequence behind its group's prefix; before, behind: sequences of no
        group, with the first and last of `own`."""
        n = before + sum(groups) + behind
        assert len(own) == n and len(prefix) == len(groups)
        self.seqs = [before + sum(groups[:g]) for g in range(len(groups) + 1)]
        self.first, self.shared = list(range(n)), [0] * n
        for g, p in enumerate(prefix):
            for i in range(self.seqs[g], self.seqs[g + 1]):
                self.first[i], self.shared[i] = self.seqs[g], p
        kv = [a + b for a, b in zip(own, self.shared)]
        hq, hkv, dim, page = heads
        self.cache = cache
        self.c = c = Case(hq, hkv, dim, page, dtype, kv, seed=seed) if cache is None else Case8(hq, hkv, dim, page, dtype, cache, kv, seed=seed)
        for i in range(n):
            if self.first[i] != i:
                at = self.shared[i] // page
                if kv[i] > at * page:
                    p = int(c.table[i, at])
                    for x in (c.kc, c.vc):
                        x.view(torch.int16 if cache is None else torch.int8)[p, :, : self.shared[i] % page] = -1
                    if cache is not None:
                        c.ks[p, :, : self.shared[i] % page] = math.nan
                        c.vs[p, :, : self.shared[i] % page] = math.inf
                c.table[i, :at] = 1 << 30
        self.prefix = prefix

    def run(self, q, out, max_len=0, max_prefix=0, seqs=None, prefix=None, kv=None, table=None):
        c = self.c
        b = qe_mixer.Batch(ints(kv or c.kv_len), c.table if table is None else table, max_len=max_len)
        sh = qe_mixer.Shared(ints(seqs or self.seqs), ints(prefix or self.prefix), max_prefix)
        if self.cache is None:
            c.att.decode_shared(b, sh, q, c.kc, c.vc, out)
        else:
            c.att.decode8_shared(b, sh, q, c.cache(), out)

    def expect(self, q):
        c = self.c
        out, off = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
        cache = ((c.kc, None), (c.vc, None)) if self.cache is None else ((c.kc, c.ks), (c.vc, c.vs))
        for i, n in enumerate(c.kv_len):
            for h in range(c.hkv):
                k, v = Q.rows_of(c, cache, i, h, n, self.first[i], self.shared[i])
                j = slice(h * (c.hq // c.hkv), (h + 1) * (c.hq // c.hkv))
                place = torch.full((c.hq // c.hkv,), n - 1, device="cuda")
                out[i, j], off[i, j] = (R if self.cache is None else Q).attend(q[i, j], k, v, place, c.dim ** -0.5)
        return out, off


def close(out, want, off):
    assert torch.isfinite(out).all()
    d = (out.double() - want).abs()
    assert bool((d <= off).all()), float((d / off).max())


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", HEADS)
def test_groups_of_all_kinds(heads, dtype, cache):
    """Sequences of no group before and behind, a group without a prefix, one without sequences, own parts of no and of one
    position, prefixes that end in any place of a page and of a step."""
    groups, prefix = [3, 0, 1, 9, 2, 4], [70, 40, 333, 257, 0, 16]
    own = [5, 1, 0, 33] + [64, 3, 200, 1, 2, 15, 16, 17, 31, 100] + [40, 0] + [7, 300, 0, 32] + [29]
    g = Grouped(heads, dtype, cache, groups, own, prefix, before=1, behind=1)
    q = g.c.q(len(own))
    want, off = g.expect(q)
    for hints in ((0, 0), (max(g.c.kv_len), max(prefix)), (1, 1)):
        out = torch.full_like(q, 7.0)
        g.run(q, out, *hints)
        g.c.att.check()
        close(out, want, off)
    assert bool((out[15] == 0).all())  # no position at all


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("heads,n,prefix", [((16, 2, 256, 256), 32, 5000), ((32, 8, 128, 64), 40, 3001), ((24, 8, 64, 16), 70, 2000), ((8, 1, 256, 16), 3, 9000)])
def test_long_prefixes(heads, n, prefix, cache):
    own = [1 + 37 * i * i % 700 for i in range(n)]
    g = Grouped(heads, torch.bfloat16, cache, [n], own, [prefix])
    q = g.c.q(n)
    want, off = g.expect(q)
    for hints in ((0, 0), (max(g.c.kv_len), prefix)):
        out = torch.empty_like(q)
        g.run(q, out, *hints)
        close(out, want, off)
    g.run(q, q, max(g.c.kv_len), prefix)  # in place
    close(q, want, off)
    g.c.att.check()


@pytest.mark.parametrize("cache", [None, torch.int8])
def test_more_rows_than_a_launch_takes(cache):
    """2^15 rows are a launch's: groups that reach over its end are in both."""
    heads, n = (256, 16, 64, 16), 300  # 128 sequences a launch
    own = [1 + 7 * i % 40 for i in range(n)]
    g = Grouped(heads, torch.float16, cache, [100, 50, 149], own, [50, 33, 90], behind=1)
    q = g.c.q(n)
    out = torch.empty_like(q)
    g.run(q, out)
    g.c.att.check()
    close(out, *g.expect(q))


def test_as_the_plain_call():
    """On tables with the shared pages in them, the results are those of decode, but for rounding."""
    g = Grouped((16, 2, 256, 64), torch.bfloat16, None, [6], [3, 50, 64, 1, 700, 9], [640])
    c = g.c
    q = c.q(6)
    one, two = torch.empty_like(q), torch.empty_like(q)
    g.run(q, one)
    c.table[1:, :10] = c.table[0, :10]
    c.att.decode(c.batch(), q, c.kc, c.vc, two)
    want, off = g.expect(q)
    close(one, want, off)
    close(two, want, off)


@pytest.mark.parametrize("cache", [None, torch.int8])
def test_values_that_are_not_finite(cache):
    """Among the shared positions they reach the group, among a sequence's own that sequence."""
    for place, hit in (((0, 20), [0, 1, 2]), ((1, 110), [1]), ((3, 4), [3, 4])):
        g = Grouped((4, 2, 64, 16), torch.bfloat16, cache, [3, 2], [20, 30, 40, 5, 6], [100, 50])
        c = g.c
        q = c.q(5)
        want, off = g.expect(q)
        p, r = int(c.table[place[0], place[1] // 16]), place[1] % 16
        if cache is None:
            c.vc[p, 1, r, 7] = math.nan
        else:
            c.vs[p, 1, r] = math.nan
        out = torch.empty_like(q)
        g.run(q, out)
        gone = torch.zeros(5, 4, dtype=torch.bool, device="cuda")
        gone[hit, 2:] = True
        assert bool(torch.isnan(out[gone][:, 7]).all())
        close(out[~gone], want[~gone], off[~gone])


@pytest.mark.parametrize("cache", [None, torch.float8_e4m3fn])
def test_bad_values_give_zeros_and_an_error(cache):
    g = Grouped((8, 2, 64, 32), torch.float16, cache, [3, 2], [20, 30, 40, 5, 66], [100, 500], behind=0)
    c = g.c
    q = c.q(5)
    want, off = g.expect(q)

    def tried(word, lost, **kw):
        out = torch.full_like(q, 7.0)
        g.run(q, out, **kw)
        with pytest.raises(qe_moe.QeError, match=word):
            c.att.check()
        rest = [i for i in range(5) if i not in lost]
        assert bool((out[lost] == 0).all()), kw
        close(out[rest], want[rest], off[rest])

    for wrong in (-1, c.kc.shape[0], (1 << 31) - 1):
        for at, lost in (((0, 1), [0, 1, 2]), ((0, 3), [0, 1, 2]), ((3, 15), [3, 4]), ((1, 4), [1]), ((4, 17), [4])):
            table = c.table.clone()
            table[at] = wrong
            tried("page", lost, table=table)
    most = c.table.shape[1] * 32
    for i in range(5):
        for wrong in (-1, most + 1, g.shared[i] - 1, (1 << 31) - 1, -(1 << 31)):
            kv = list(c.kv_len)
            kv[i] = wrong
            tried("length", [i], kv=kv)
    for wrong in (-1, most + 1, (1 << 31) - 1):
        tried("length", [0, 1, 2], prefix=[wrong, 500])
    tried("offset", [0, 1, 2], seqs=[-1, 3, 5])
    tried("offset", [3, 4], seqs=[0, 3, 6])
    tried("offset", [3, 4], seqs=[0, 3, (1 << 31) - 1])
    for seqs in ([0, 5, 3], [3, 0, 5], [0, 4, 1]):  # falling: reported, whatever the outputs hold
        g.run(q, torch.empty_like(q), seqs=seqs)
        with pytest.raises(qe_moe.QeError, match="offset"):
            c.att.check()
    out = torch.empty_like(q)
    g.run(q, out)
    c.att.check()
    close(out, want, off)


def test_refusals():
    g = Grouped((8, 2, 64, 32), torch.float16, None, [2], [5, 9], [40])
    c = g.c
    q = c.q(2)
    out, a = torch.empty_like(q), c.att
    sh = qe_mixer.Shared(ints([0, 2]), ints([40]))
    with pytest.raises(qe_moe.QeError, match="cu_q"):
        a.decode_shared(c.batch([0, 1, 2]), sh, q, c.kc, c.vc, out)
    for bad in (dict(q=q.float()), dict(out=out.bfloat16()), dict(kc=c.kc.float()), dict(vc=c.vc[1:])):
        with pytest.raises(ValueError):
            a.decode_shared(c.batch(), sh, **{**dict(q=q, kc=c.kc, vc=c.vc, out=out), **bad})
    for seqs, prefix in ((ints([0, 2]).long(), ints([40])), (ints([0, 2]), ints([40, 3])), (ints([0, 2]).cpu(), ints([40]))):
        with pytest.raises(ValueError):
            qe_mixer.Shared(seqs, prefix)
    with pytest.raises(ValueError):
        a.decode_shared(c.batch(), qe_mixer.Shared(ints([0, 2]).cpu(), ints([40]).cpu()), q, c.kc, c.vc, out)
    for field, value, word in (("n_groups", 0, "n_groups"), ("n_groups", 65536, "n_groups"), ("seqs", None, "null"), ("prefix", None, "null"), ("max_prefix", -1, "max_prefix")):
        sh = qe_mixer.Shared(ints([0, 2]), ints([40]))
        setattr(sh.c, field, value)
        with pytest.raises(qe_moe.QeError, match=word):
            a.decode_shared(c.batch(), sh, q, c.kc, c.vc, out)
    a.check()
