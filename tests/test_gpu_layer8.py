"""A server's attention layer over an 8-bit cache, call after call: a system prompt, questions behind it, answers token by token."""
import math

import pytest

torch = pytest.importorskip("torch")
import cache8_ref as Q  # noqa: E402
import qe_mixer  # noqa: E402
import qe_moe  # noqa: E402
from cache8_ref import gen, ints, rand, same  # noqa: E402

pytestmark = pytest.mark.gpu


class Server:
    """Three conversations behind one system prompt: their tables' first pages are the first one's."""

    def __init__(self, codes, dtype, hq, hkv, dim, page, system, seed=0):
        self.g = gen(seed)
        self.n, self.page, self.dim, self.hq, self.hkv, self.dtype, self.system = 3, page, dim, hq, hkv, dtype, system
        cols = -(-(system + 200) // page)
        self.table = torch.randperm(self.n * cols, generator=self.g, device="cuda").to(torch.int32).view(self.n, cols)
        shape = (self.n * cols, hkv, page, dim)
        self.cache = qe_mixer.Cache8(*(torch.zeros(shape, dtype=codes, device="cuda") for _ in range(2)), *(torch.zeros(shape[:3], device="cuda") for _ in range(2)))
        self.att = qe_mixer.Attention(hq, hkv, dim, page, dtype=dtype, rotary=dim // 2, theta=1e6)
        self.norms = qe_mixer.Norms(1 + rand(self.g, dim, std=0.2), 1 + rand(self.g, dim, std=0.2))
        self.kv_len = torch.zeros(self.n, dtype=torch.int32, device="cuda")
        self.shared = qe_mixer.Shared(ints([0, self.n]), ints([system]), system)
        # the page that the system prompt ends in is copied to the others before they go on in it
        self.whole = system // page

    def rows(self, T):
        return rand(self.g, T, self.hq + 2 * self.hkv, self.dim, std=2.0).split((self.hq, self.hkv, self.hkv), 1)

    def values(self, i):
        """Keys and values of conversation i as the cache has them, in 64 bits."""
        n = int(self.kv_len[i])
        at = torch.arange(n, device="cuda")
        rows = torch.where(at < self.system, 0, i)
        p = self.table[rows, at // self.page].long()
        out = []
        for c, s in ((self.cache.kc, self.cache.k_scale), (self.cache.vc, self.cache.v_scale)):
            out.append(Q.values(c.view(torch.int8)[p, :, at % self.page].view(c.dtype), s[p, :, at % self.page]))
        return out

    def expect(self, q, i):
        """Rows q of conversation i's last positions."""
        k, v = self.values(i)
        place = torch.arange(k.shape[0] - q.shape[0], k.shape[0], device="cuda")
        group = self.hq // self.hkv
        pairs = [Q.attend(q[:, h], k[:, h // group], v[:, h // group], place, self.dim ** -0.5) for h in range(self.hq)]
        return [torch.stack(x, 1) for x in zip(*pairs)]


def close(out, want, off):
    assert torch.isfinite(out).all()
    assert bool(((out.double() - want).abs() <= off).all()), float(((out.double() - want).abs() / off).max())


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype,hq,hkv,dim,page,system", [(torch.bfloat16, 16, 2, 256, 64, 150), (torch.float16, 8, 4, 128, 32, 96), (torch.bfloat16, 6, 1, 64, 16, 77)])
def test_conversations(codes, dtype, hq, hkv, dim, page, system):
    s = Server(codes, dtype, hq, hkv, dim, page, system)
    # the system prompt, into the first one's pages
    q, k, v = s.rows(system)
    rot, out = (torch.empty(system, hq, dim, dtype=dtype, device="cuda") for _ in range(2))
    s.kv_len[0] = system
    b = qe_mixer.Batch(s.kv_len[:1], s.table[:1], ints([0, system]))
    s.att.append8(b, q, k, v, s.cache, rot, norms=s.norms)
    s.att.prompt8(b, rot, s.cache, out)
    close(out, *s.expect(rot, 0))
    # read back, it is what 16 bits of it would be
    kb, vb = (torch.empty(system, hkv, dim, dtype=dtype, device="cuda") for _ in range(2))
    s.att.read8(b, s.cache, kb, vb)
    for got, want in zip((kb, vb), s.values(0)):
        assert bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + 1e-7).all())
    # questions of three lengths: tokens of their own behind it, which prompt8 sees through tables with the shared pages
    lens = [30, 1, 45]
    s.table[1:, : s.whole] = s.table[0, : s.whole]
    if system % page:
        for x in (s.cache.kc, s.cache.vc, s.cache.k_scale, s.cache.v_scale):
            x.view(torch.int8)[s.table[1:, s.whole].long()] = x.view(torch.int8)[s.table[0, s.whole].long()].clone()
    s.kv_len.copy_(ints([system + x for x in lens]))
    T = sum(lens)
    q, k, v = s.rows(T)
    rot, out = (torch.empty(T, hq, dim, dtype=dtype, device="cuda") for _ in range(2))
    b = qe_mixer.Batch(s.kv_len, s.table, ints([0, 30, 31, 76]))
    s.att.append8(b, q, k, v, s.cache, rot, norms=s.norms)
    s.att.prompt8(b, rot, s.cache, out)
    for i, (x, y) in enumerate(((0, 30), (30, 31), (31, 76))):
        close(out[x:y], *s.expect(rot[x:y], i))
    # answers, token by token: both single-token calls, captured once and replayed
    one = qe_mixer.Batch(s.kv_len, s.table, max_len=system + 200)
    q, k, v = (torch.empty(3, h, dim, device="cuda") for h in (hq, hkv, hkv))
    rot, plain, shared = (torch.zeros(3, hq, dim, dtype=dtype, device="cuda") for _ in range(3))

    def step(stream=None):
        s.att.append8(one, q, k, v, s.cache, rot, norms=s.norms, stream=stream)
        s.att.decode8(one, rot, s.cache, plain, stream=stream)
        s.att.decode8_shared(one, s.shared, rot, s.cache, shared, stream=stream)

    def token(run):
        s.kv_len += 1
        for x in (q, k, v):
            x.copy_(rand(s.g, *x.shape, std=2.0))
        run()
        for i in range(3):
            want, off = s.expect(rot[i: i + 1], i)
            close(plain[i: i + 1], want, off)
            close(shared[i: i + 1], want, off)

    token(step)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream())
    for i in range(4):
        token(graph.replay)
        if i == 1:
            token(step)  # eager work between replays
    s.att.check()


def test_16_bit_norms_and_shared_beginnings_together():
    """append with norms, prompt and both single-token calls over a 16-bit cache."""
    g = gen(5)
    hq, hkv, dim, page, n = 16, 2, 128, 32, 4
    att = qe_mixer.Attention(hq, hkv, dim, page, rotary=128, theta=1e4)
    norms = qe_mixer.Norms(1 + rand(g, dim, std=0.2), 1 + rand(g, dim, std=0.2))
    kc, vc = (torch.zeros(40, hkv, page, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.arange(40, device="cuda", dtype=torch.int32).view(n, 10).contiguous()
    table[1:, :4] = table[0, :4]  # 128 shared positions
    kv = torch.tensor([128, 0, 0, 0], dtype=torch.int32, device="cuda")
    q, k, v = rand(g, 128, hq + 2 * hkv, dim, dtype=torch.bfloat16).split((hq, hkv, hkv), 1)
    rot, out = torch.empty(128, hq, dim, dtype=torch.bfloat16, device="cuda"), torch.empty(128, hq, dim, dtype=torch.bfloat16, device="cuda")
    b = qe_mixer.Batch(kv, table, ints([0, 128, 128, 128, 128]))
    att.append(b, q, k, v, kc, vc, rot, norms=norms)
    att.prompt(b, rot, kc, vc, out)
    kv.copy_(ints([128, 128, 128, 128]))
    one = qe_mixer.Batch(kv, table)
    shared = qe_mixer.Shared(ints([0, 4]), ints([128]))
    for _ in range(3):
        kv += 1
        q, k, v = rand(g, n, hq + 2 * hkv, dim, dtype=torch.bfloat16).split((hq, hkv, hkv), 1)
        rot, x, y = (torch.empty(n, hq, dim, dtype=torch.bfloat16, device="cuda") for _ in range(3))
        att.append(one, q, k, v, kc, vc, rot, norms=norms)
        att.decode(one, rot, kc, vc, x)
        att.decode_shared(one, shared, rot, kc, vc, y)
        # two roundings of each, and of their probabilities, apart
        assert bool(((x.float() - y.float()).abs() <= 2.0 ** -6 * (x.float().abs() + 1)).all())
    att.check()


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_results_do_not_change_from_call_to_call(codes):
    c = Q.Case8(16, 2, 128, 32, torch.bfloat16, codes, [5000, 700, 3, 90])
    one, many = c.batch(), c.batch([0, 40, 300, 303, 333])
    sh = qe_mixer.Shared(ints([0, 2, 4]), ints([600, 3]))
    q, p = c.q(4), c.q(333)

    def run():
        outs = [torch.empty_like(q), torch.empty_like(q), torch.empty_like(p)]
        c.att.decode8(one, q, c.cache(), outs[0])
        c.att.decode8_shared(one, sh, q, c.cache(), outs[1])
        c.att.prompt8(many, p, c.cache(), outs[2])
        return outs

    first = run()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))
    c.att.check()


def test_contexts_on_streams_of_their_own():
    cases = [Q.Case8(8, 2, 64, 16, torch.float16, torch.int8, [3000, 50], seed=i) for i in range(2)]
    q = [c.q(2) for c in cases]
    sh = qe_mixer.Shared(ints([0, 2]), ints([40]))
    want = []
    for c, x in zip(cases, q):
        o = torch.empty_like(x)
        c.att.decode8_shared(c.batch(), sh, x, c.cache(), o)
        want.append(o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[torch.empty_like(x) for _ in range(20)] for x in q]
    batches, caches = [c.batch() for c in cases], [c.cache() for c in cases]
    torch.cuda.synchronize()
    for r in range(20):
        for i, c in enumerate(cases):
            c.att.decode8_shared(batches[i], sh, q[i], caches[i], outs[i][r], stream=streams[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])
        cases[i].att.check()


def test_two_graphs_share_a_context():
    c = Q.Case8(8, 2, 128, 32, torch.bfloat16, torch.int8, [2000, 90, 900])
    q = c.q(3)
    sh = qe_mixer.Shared(ints([0, 3]), ints([80]), 80)
    b, cache = c.batch(), c.cache()
    want = [torch.empty_like(q) for _ in range(2)]
    c.att.decode8(b, q, cache, want[0])
    c.att.decode8_shared(b, sh, q, cache, want[1])
    outs = [torch.zeros_like(q) for _ in range(2)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    torch.cuda.synchronize()
    for i, call in enumerate((lambda st: c.att.decode8(b, q, cache, outs[0], stream=st), lambda st: c.att.decode8_shared(b, sh, q, cache, outs[1], stream=st))):
        with torch.cuda.graph(graphs[i]):
            call(torch.cuda.current_stream())
    for _ in range(3):
        for i in (0, 1):
            outs[i].zero_()
            graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    c.att.check()


def test_more_threads_than_a_launch_has_are_refused():
    n = 65535
    att = qe_mixer.Attention(256, 256, 64, 16)
    zeros = torch.zeros(n, dtype=torch.int32, device="cuda")
    pages = torch.zeros(1, 256, 16, 64, dtype=torch.int8, device="cuda")
    cache = qe_mixer.Cache8(pages, pages.clone(), torch.zeros(1, 256, 16, device="cuda"), torch.zeros(1, 256, 16, device="cuda"))
    rows = torch.zeros(256, 256, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(qe_moe.QeError, match="threads"):
        att.prompt8(qe_mixer.Batch(zeros, zeros[:, None].contiguous(), torch.zeros(n + 1, dtype=torch.int32, device="cuda")), rows, cache, torch.empty_like(rows))
    b = qe_mixer.Batch(zeros[:256], zeros[:256, None].contiguous())
    with pytest.raises(qe_moe.QeError, match="threads"):
        att.decode8_shared(b, qe_mixer.Shared(torch.zeros(n + 1, dtype=torch.int32, device="cuda"), zeros), rows, cache, torch.empty_like(rows))
    att.check()


def test_rows_of_another_type_are_refused():
    """Rows of 16 bits for another type's context are refused, not read as if they were its."""
    c = Q.Case8(4, 2, 64, 16, torch.float16, torch.int8, [9])
    cache, before = c.copy(), c.copy()
    k = rand(c.g, 9, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        c.att.append8(c.batch([0, 9]), None, k, k, cache, None)
    with pytest.raises(ValueError):
        c.att.read8(c.batch([0, 9]), cache, k, None)
    assert same(cache, before) and math.isfinite(float(k.float().sum()))
