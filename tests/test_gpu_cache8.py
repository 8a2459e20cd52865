"""Norms with the rotation, the write to an 8-bit cache and its read, against their definitions in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
import cache8_ref as Q  # noqa: E402
import mixer_ref as R  # noqa: E402
import qe_mixer  # noqa: E402
import qe_moe  # noqa: E402
from cache8_ref import Case8, bits, gen, ints, rand, same  # noqa: E402

pytestmark = pytest.mark.gpu
EPS = 1e-6
GEOMETRIES = [(16, 2, 256, 256, 64, (11, 11, 10), True), (4, 2, 128, 16, 128, (64,), False), (3, 3, 64, 32, 48, (10, 8, 6), False),
              (40, 8, 64, 16, 64, (14, 9, 9), True), (2, 2, 64, 16, 0, (0,), False)]


@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn, None])  # None: a 16-bit cache
@pytest.mark.parametrize("dtype,in_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("hq,hkv,dim,page,rotary,sections,interleaved", GEOMETRIES)
def test_append(hq, hkv, dim, page, rotary, sections, interleaved, dtype, in_dtype, codes, normed):
    if codes is None and not normed:
        pytest.skip("that is the append without norms")
    lens, kv = [1, 40, 0, 3], [1, 140, 7, 64]
    c = Case8(hq, hkv, dim, page, dtype, codes or torch.int8, kv, rotary=rotary, theta=1e7, sections=sections, interleaved=interleaved)
    T = sum(lens)
    q, k, v = rand(c.g, T + 2, hq + 2 * hkv, dim, dtype=in_dtype, std=3.0).split((hq, hkv, hkv), 1)
    wq, wk = (1 + rand(c.g, dim, std=0.3) for _ in range(2))
    norms = qe_mixer.Norms(wq, wk, EPS) if normed else None
    pos = torch.randint(0, 262144, (len(sections), T + 2), generator=c.g, device="cuda").to(torch.int32)
    cu = [0, 1, 41, 41, 44]
    out = torch.full((T + 2, hq, dim), 7.0, dtype=dtype, device="cuda")
    b = c.batch(cu)
    if codes is None:
        kc, vc = (rand(c.g, c.kc.shape[0], hkv, page, dim, dtype=dtype) for _ in range(2))
        kept = kc.clone(), vc.clone()
        c.att.append(b, q, k, v, kc, vc, out, pos=pos, norms=norms)
    else:
        cache = c.copy()
        kc, vc, kept = cache.kc, cache.vc, (c.kc, c.vc, c.ks, c.vs)
        c.att.append8(b, q, k, v, cache, out, pos=pos, norms=norms)
    c.att.check()
    axes = R.axes_of(rotary, sections, interleaved)

    def expect(x, w):
        y, off = Q.norm(x, w if normed else None, EPS)
        z, turned = R.rotate(y, pos, rotary, 1e7, axes)
        _, more = R.rotate(off * 2.0 ** 21, pos, rotary, 1e7, axes)  # |a| + |b| of the offsets, in rotated places
        return z, turned + torch.maximum(off, more)

    u = R.U[dtype]
    want, off = expect(q, wq)
    assert bool(((out[:T].double().cpu() - want[:T]).abs() <= off[:T] + u * want[:T].abs() + 1e-7).all())
    assert bool((out[T:] == 7).all())
    places = [(int(c.table[i, (kv[i] - n + j) // page]), (kv[i] - n + j) % page) for i, n in enumerate(lens) for j in range(n)]
    p, r = (torch.tensor(x, device="cuda") for x in zip(*places))
    want, off = expect(k, wk)
    if codes is None:
        assert bool(((kc[p, :, r].double().cpu() - want[:T]).abs() <= off[:T] + u * want[:T].abs() + 1e-7).all())
        assert torch.equal(vc[p, :, r], v[:T].to(dtype))
        pairs = ((kc, kept[0]), (vc, kept[1]))
    else:
        Q.stored_rows(want[:T].reshape(-1, dim), off[:T].reshape(-1, dim), kc[p, :, r].reshape(-1, dim), cache.k_scale[p, :, r].reshape(-1))
        plain = v[:T].double().reshape(-1, dim)
        Q.stored_rows(plain, torch.zeros_like(plain), vc[p, :, r].reshape(-1, dim), cache.v_scale[p, :, r].reshape(-1))
        pairs = ((kc, kept[0]), (vc, kept[1]), (cache.k_scale, kept[2]), (cache.v_scale, kept[3]))
    for new, old in pairs:  # nothing else was written
        rest = torch.ones(new.shape[0], page, dtype=torch.bool, device="cuda")
        rest[p, r] = False
        assert torch.equal(bits(new).transpose(1, 2)[rest], bits(old).transpose(1, 2)[rest])


@pytest.mark.parametrize("which", ["q", "k"])
def test_append_norms_only_one(which):
    c = Case8(4, 2, 128, 32, torch.float16, torch.int8, [50], rotary=64)
    q, k, v = (rand(c.g, 9, h, 128, dtype=torch.float16) for h in (4, 2, 2))
    w = 1 + rand(c.g, 128, std=0.3)
    out, both, none = (torch.empty_like(q) for _ in range(3))
    one, normed, plain = c.copy(), c.copy(), c.copy()
    c.att.append8(c.batch([0, 9]), q, k, v, one, out, norms=qe_mixer.Norms(*((w, None) if which == "q" else (None, w))))
    c.att.append8(c.batch([0, 9]), q, k, v, normed, both, norms=qe_mixer.Norms(w, w))
    c.att.append8(c.batch([0, 9]), q, k, v, plain, none)
    assert torch.equal(out, both if which == "q" else none)
    assert same(one, plain if which == "q" else normed)


def test_append_in_place_without_q_and_of_single_tokens():
    c = Case8(14, 2, 128, 32, torch.bfloat16, torch.float8_e4m3fn, [50, 33, 1], rotary=128)
    q, k, v = (rand(c.g, 3, h, 128, dtype=torch.bfloat16) for h in (14, 2, 2))
    norms = qe_mixer.Norms(1 + rand(c.g, 128, std=0.3), 1 + rand(c.g, 128, std=0.3), 1e-5)
    out, one, two, three = torch.empty_like(q), c.copy(), c.copy(), c.copy()
    c.att.append8(c.batch(), q, k, v, one, out, norms=norms)
    c.att.append8(c.batch(), None, k, v, two, None, norms=norms)
    c.att.append8(c.batch([0, 1, 2, 3]), q, k, v, three, q, pos=ints([[49, 32, 0]]), norms=norms)
    c.att.check()
    assert torch.equal(out, q) and same(one, two) and same(one, three) and not same(one, c.cache())


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("in_dtype", [torch.float32, torch.bfloat16])
def test_rows_of_zeros_tiny_huge_and_not_finite(codes, in_dtype):
    c = Case8(2, 1, 64, 16, torch.bfloat16, codes, [7])
    x = rand(c.g, 7, 1, 64, dtype=in_dtype)
    x[0] = 0
    x[1] *= 2.0 ** -110  # below 2^-100: zeros
    x[2] *= 2.0 ** -90
    x[3] *= 2.0 ** 120
    x[4, 0, 5] = math.inf
    x[5, 0, 63] = math.nan
    x[6, 0, 17] = -math.inf
    cache, back = c.copy(), torch.empty(7, 1, 64, dtype=torch.bfloat16, device="cuda")
    c.att.append8(c.batch([0, 7]), None, x, x, cache, None)
    p = int(c.table[0, 0])
    for cc, s in ((cache.kc, cache.k_scale), (cache.vc, cache.v_scale)):
        assert bool((s[p, 0, :2] == 0).all()) and bool((cc[p, 0, :2].float() == 0).all())
        Q.stored_rows(x[2:4, 0].double(), torch.zeros(2, 64), cc[p, 0, 2:4], s[p, 0, 2:4])
        assert bool(torch.isnan(s[p, 0, 4:7]).all())
    c.att.read8(c.batch([0, 7]), cache, back, None)
    c.att.check()
    assert bool((back[:2] == 0).all()) and bool(torch.isnan(back[4:]).all()) and bool(torch.isfinite(back[:4]).all())
    # norms: a row of zeros stays one, squares beyond 32 bits are NaN
    w = torch.ones(64, device="cuda")
    c.att.append8(c.batch([0, 7]), None, x, x, cache, None, norms=qe_mixer.Norms(None, w))
    c.att.read8(c.batch([0, 7]), cache, back, None)
    assert bool((back[0] == 0).all()) and bool(torch.isnan(back[3:]).all()) and bool(torch.isfinite(back[:3]).all())


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hkv,dim,page", [(2, 256, 256), (8, 128, 64), (3, 64, 16), (1, 64, 32), (1, 256, 16)])
def test_read(hkv, dim, page, dtype, codes):
    kv = [700, 1, 0, 65, 300]
    c = Case8(hkv, hkv, dim, page, dtype, codes, kv)
    lens = [700, 1, 0, 30, 300]
    cu = [0, 700, 701, 701, 731, 1031]
    wide = torch.full((1033, 2 * hkv + 1, dim), 7.0, dtype=dtype, device="cuda")
    k, v = wide[:, :hkv], wide[:, hkv: 2 * hkv]
    c.att.read8(c.batch(cu), c.cache(), k, v)
    c.att.check()
    for i, n in enumerate(lens):
        at = torch.arange(kv[i] - n, kv[i], device="cuda")
        p, r = c.table[i, at // page].long(), at % page
        for got, cc, s in ((k, c.kc, c.ks), (v, c.vc, c.vs)):
            want = (cc.view(torch.int8)[p, :, r].view(codes).float() * s[p, :, r][..., None]).to(dtype)
            assert torch.equal(got[cu[i]: cu[i + 1]], want)
    assert bool((wide[1031:] == 7).all()) and bool((wide[:, 2 * hkv] == 7).all())
    # single tokens, and one of the two
    one = torch.empty(5, hkv, dim, dtype=dtype, device="cuda")
    kv[2] = 3
    c.table[2, 0] = 0
    b = qe_mixer.Batch(ints(kv), c.table)
    c.att.read8(b, c.cache(), None, one)
    assert torch.equal(one[0], v[699]) and torch.equal(one[4], v[1030])
    c.att.check()


def test_bad_lengths_pages_and_offsets():
    c = Case8(2, 2, 64, 16, torch.float16, torch.int8, [40, 60, 20], rotary=64)
    k = rand(c.g, 50, 2, 64, dtype=torch.float16)
    norms = qe_mixer.Norms(torch.ones(64, device="cuda"), torch.ones(64, device="cuda"))
    want_k, want_v = (torch.empty_like(k) for _ in range(2))
    c.att.read8(c.batch([0, 20, 40, 50]), c.cache(), want_k, want_v)

    def tried(b, word, lost):
        rot, back = torch.full_like(k, 7.0), torch.full_like(k, 7.0)
        cache = c.copy()
        c.att.append8(b, k, k, k, cache, rot, norms=norms)
        with pytest.raises(qe_moe.QeError, match=word):
            c.att.check()
        c.att.read8(b, c.cache(), back, None)
        with pytest.raises(qe_moe.QeError, match=word):
            c.att.check()
        gone = torch.zeros(50, dtype=torch.bool, device="cuda")
        for x, y in lost:
            gone[x:y] = True
        assert bool((back[gone] == 0).all()) and torch.equal(back[~gone], want_k[~gone])
        assert bool((rot[gone] == 7).all()) and not bool((rot[~gone] == 7).any())
        return cache

    for wrong in (-1, c.table.shape[1] * 16 + 1, (1 << 31) - 1, -(1 << 31)):
        tried(qe_mixer.Batch(ints([40, wrong, 20]), c.table, ints([0, 20, 40, 50])), "length", [(20, 40)])
    for wrong in (-1, c.kc.shape[0], (1 << 31) - 1):
        table = c.table.clone()
        table[0, 2] = wrong  # positions 32 to 39 of the last 20
        tried(qe_mixer.Batch(ints([40, 60, 20]), table, ints([0, 20, 40, 50])), "page", [(12, 20)])
    tried(c.batch([0, 20, 40, 51]), "offset", [(40, 50)])
    tried(c.batch([-3, 20, 40, 50]), "offset", [(0, 20)])
    tried(c.batch([0, 50, 40, 50]), "offset", [(0, 50)])
    assert same(tried(c.batch([0, 50, 40, 50]), "offset", [(0, 50)]), c.cache())  # nothing of those was written
    # before the first position: no page is touched, a read gives zeros
    cache, back = c.copy(), torch.full_like(k, 7.0)
    b = qe_mixer.Batch(ints([2, 0, 20]), c.table, ints([0, 20, 40, 50]))
    c.att.read8(b, c.cache(), back, None)
    c.att.append8(b, None, k, k, cache, None)
    c.att.check()
    assert bool((back[:18] == 0).all()) and bool((back[20:40] == 0).all()) and torch.equal(back[40:], want_k[40:])
    cache.kc[int(c.table[0, 0]), :, :2] = c.kc[int(c.table[0, 0]), :, :2]
    p = c.table[2, 0].long(), c.table[2, 1].long()
    for x in p:
        cache.kc[x] = c.kc[x]
    assert torch.equal(cache.kc, c.kc)


def test_more_sequences_than_threads_report_their_offsets():
    n = 700
    c = Case8(1, 1, 64, 16, torch.float16, torch.int8, [20, 3] + [0] * (n - 2))
    k = rand(c.g, 2, 1, 64, dtype=torch.float16)
    for at, what in ((n, 3), (n - 1, 5), (n - 100, 1), (400, -1)):
        cu = [0, 1] + [2] * (n - 1)
        cu[at] = what
        for call in (lambda: c.att.append8(c.batch(cu), None, k, k, c.copy(), None), lambda: c.att.read8(c.batch(cu), c.cache(), k.clone(), None)):
            call()
            with pytest.raises(qe_moe.QeError, match="offset"):
                c.att.check()


def test_far_offsets_in_a_large_cache():
    """Pages whose codes start past 2^32 bytes."""
    hkv, dim, page = 2, 256, 256
    pages = (1 << 32) // (hkv * page * dim) + 40
    kc, vc = (torch.empty(pages, hkv, page, dim, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(pages, hkv, page, device="cuda") for _ in range(2))
    cache = qe_mixer.Cache8(kc, vc, ks, vs)
    table = ints([[5, pages - 7], [pages - 1, 0]])
    g = gen(3)
    att = qe_mixer.Attention(16, hkv, dim, page)
    k, v = rand(g, 2, hkv, dim), rand(g, 2, hkv, dim)
    back = [torch.empty(2, hkv, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    b = qe_mixer.Batch(ints([400, 256]), table)
    att.append8(b, None, k, v, cache, None)
    att.read8(b, cache, *back)
    att.check()
    for i, (p, r) in enumerate(((pages - 7, 143), (pages - 1, 255))):
        for x, cc, s, y in ((k, kc, ks, back[0]), (v, vc, vs, back[1])):
            Q.stored_rows(x[i].double(), torch.zeros(hkv, dim), cc[p, :, r], s[p, :, r])
            assert torch.equal(y[i], (cc[p, :, r].float() * s[p, :, r][:, None]).bfloat16())


def test_refusals():
    c = Case8(8, 2, 64, 32, torch.float16, torch.int8, [50, 60], rotary=64)
    q, k = c.q(2), rand(c.g, 2, 2, 64, dtype=torch.float16)
    out, a, w = torch.empty_like(q), c.att, torch.ones(64, device="cuda")
    for bad in (dict(kc=c.kc.float()), dict(vc=c.vc[1:]), dict(kc=c.kc.transpose(1, 2)), dict(vc=c.vc.view(torch.uint8)), dict(k_scale=c.ks.half()),
                dict(k_scale=c.ks[1:]), dict(v_scale=c.vs.cpu()), dict(kc=c.kc.cpu())):
        with pytest.raises(ValueError):
            qe_mixer.Cache8(**{**dict(kc=c.kc, vc=c.vc, k_scale=c.ks, v_scale=c.vs), **bad})
    for bad in (dict(q_weight=w.half(), k_weight=w), dict(q_weight=w[::2], k_weight=None), dict(q_weight=w, k_weight=w[:32]), dict(q_weight=w[None], k_weight=w)):
        with pytest.raises(ValueError):
            qe_mixer.Norms(**bad)
    for norms in (qe_mixer.Norms(w[:32], None), qe_mixer.Norms(w.cpu(), w.cpu())):
        with pytest.raises(ValueError):
            a.append8(c.batch(), q, k, k, c.cache(), out, norms=norms)
    for eps in (0.0, -1.0, math.nan, math.inf, 1e-31):
        with pytest.raises(qe_moe.QeError, match="eps"):
            a.append8(c.batch(), q, k, k, c.cache(), out, norms=qe_mixer.Norms(w, w, eps))
    with pytest.raises(qe_moe.QeError, match="aligned"):
        a.append8(c.batch(), q, k, k, c.cache(), out, norms=qe_mixer.Norms(torch.ones(65, device="cuda")[1:], w))
    other = Case8(8, 4, 64, 32, torch.float16, torch.int8, [50, 60])
    with pytest.raises(ValueError):
        a.append8(c.batch(), q, k, k, other.cache(), out)
    with pytest.raises(ValueError):
        a.read8(c.batch(), c.cache(), None, None)
    with pytest.raises(ValueError):
        a.read8(c.batch(), c.cache(), k.float(), None)
    with pytest.raises(qe_moe.QeError, match="one array"):
        a.read8(c.batch(), c.cache(), k, k)
    with pytest.raises(qe_moe.QeError, match="n_tokens"):
        a.read8(c.batch(), c.cache(), c.q(3)[:, :2], None)
    cache = c.cache()
    cache.c.type = 2
    with pytest.raises(qe_moe.QeError, match="cache type"):
        a.append8(c.batch(), q, k, k, cache, out)
    a.check()
