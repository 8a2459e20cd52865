"""The gated delta rule against the recurrence in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")
import mixer_ref as R  # noqa: E402
import qe_mixer  # noqa: E402
import qe_moe  # noqa: E402

pytestmark = pytest.mark.gpu
# A result in 32 bits is a chain of at most five products of inner length up to 128 per chunk of 64 tokens, whose
# roundings add like their root: 5 sqrt(128) 2^-24 = 3.4e-6 of its size, and a state collects those of a few chunks
# before they fade.  Results in 16 bits are rounded once more.
TOL32 = 1e-5
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Case:
    def __init__(self, hk, hv, dk, dv, dtype, lens, seed=0, slots=None, rates=(1e-3, 2.0), **desc):
        g = gen(seed)
        T = sum(lens)

        def rand(*shape):
            return torch.randn(*shape, generator=g, device="cuda")

        self.dtype, self.lens, self.T = dtype, lens, T
        self.cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
        silu = torch.nn.functional.silu
        self.q, self.k, self.v = silu(rand(T, hk, dk)).to(dtype), silu(rand(T, hk, dk)).to(dtype), silu(rand(T, hv, dv)).to(dtype)
        rate = torch.exp(torch.linspace(math.log(rates[0]), math.log(rates[1]), hv, device="cuda"))
        self.g = -rate * torch.nn.functional.softplus(rand(T, hv))
        self.beta = torch.sigmoid(rand(T, hv))
        self.pool = 0.1 * rand(slots or 2 * len(lens), hv, dk, dv)
        self.out = torch.full((T, hv, dv), 7.0, dtype=dtype, device="cuda")
        self.desc = dict(l2norm=True, scale=0.0, **desc)
        self.h = qe_mixer.GatedDelta(hk, hv, dk, dv, dtype=dtype, t_max=max(T, 1), seqs_max=max(len(lens), 1), **self.desc)

    def expect(self, i, S):
        a, b = self.cu[i], self.cu[i + 1]
        return R.delta(self.q[a:b], self.k[a:b], self.v[a:b], self.g[a:b], self.beta[a:b], S, self.desc["l2norm"],
                       self.desc["scale"] or self.q.shape[2] ** -0.5)

    def close(self, out, want, what=""):
        assert torch.isfinite(out).all()
        assert R.rel(out, want) <= TOL32 + (R.U[self.dtype] if out.dtype == self.dtype != torch.float32 else 0), (what, R.rel(out, want))

    def prompt(self, slots_in, slots_out, out=None, stream=None, cu=None):
        self.h.prompt(self.q, self.k, self.v, self.g, self.beta, self.pool, ints(slots_in), ints(slots_out), ints(cu or self.cu),
                      self.out if out is None else out, stream=stream)

    def decode(self, slots_in, slots_out, out=None, stream=None):
        self.h.decode(self.q, self.k, self.v, self.g, self.beta, self.pool, ints(slots_in), ints(slots_out),
                      self.out if out is None else out, stream=stream)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hk,hv,dk,dv", [(16, 32, 128, 128), (2, 2, 64, 128), (1, 3, 128, 64), (2, 8, 64, 64)])
def test_prompt(hk, hv, dk, dv, dtype):
    lens = [1, 64, 0, 63, 65, 130, 16, 17]
    c = Case(hk, hv, dk, dv, dtype, lens)
    before = c.pool.clone()
    n = len(lens)
    into = [2 * i if i % 3 else -1 for i in range(n)]
    outof = [2 * i + 1 if i != 4 else -1 for i in range(n)]
    c.prompt(into, outof)
    c.h.check()
    for i in range(n):
        S = before[into[i]] if into[i] >= 0 else torch.zeros_like(before[0])
        o, S = c.expect(i, S)
        if lens[i]:
            c.close(c.out[c.cu[i]: c.cu[i + 1]], o, i)
        if outof[i] >= 0:
            if lens[i] == 0 and into[i] >= 0:
                assert torch.equal(c.pool[outof[i]], before[into[i]])
            c.close(c.pool[outof[i]], S, i) if lens[i] or into[i] >= 0 else None
    for s in set(range(2 * n)) - set(outof):
        assert torch.equal(c.pool[s], before[s]), s


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hk,hv,dk,dv", [(16, 32, 128, 128), (2, 2, 64, 128), (1, 3, 128, 64), (2, 8, 64, 64)])
@pytest.mark.parametrize("n", [1, 5])
def test_decode(hk, hv, dk, dv, dtype, n):
    c = Case(hk, hv, dk, dv, dtype, [1] * n)
    before = c.pool.clone()
    into = [2 * i for i in range(n)]
    into[-1] = -1
    outof = [2 * i + 1 for i in range(n)]
    outof[0] = 0  # in place
    c.decode(into, outof)
    c.h.check()
    for i in range(n):
        o, S = c.expect(i, before[into[i]] if into[i] >= 0 else torch.zeros_like(before[0]))
        c.close(c.out[i: i + 1], o, i)
        c.close(c.pool[outof[i]], S, i)
    for s in set(range(2 * n)) - set(outof):
        assert torch.equal(c.pool[s], before[s])


def test_decode_of_many_sequences():
    n = 300  # more than a workgroup looks through at once
    c = Case(1, 1, 64, 64, torch.float32, [1] * n)
    before = c.pool.clone()
    into, outof = [2 * i for i in range(n)], [2 * i + 1 for i in range(n)]
    outof[299] = 2 * 17  # what sequence 17 reads
    c.decode(into, outof)
    with pytest.raises(qe_moe.QeError, match="slot"):
        c.h.check()
    for i in (0, 17, 255, 256, 298):
        o, S = c.expect(i, before[2 * i])
        c.close(c.out[i: i + 1], o, i)
        c.close(c.pool[2 * i + 1], S, i)
    assert bool((c.out[299] == 0).all()) and torch.equal(c.pool[34], before[34])


def test_prompts_of_many_sequences():
    n = 300
    lens = [i % 4 for i in range(n)]
    lens[7], lens[299] = 130, 65
    c = Case(1, 2, 64, 64, torch.bfloat16, lens)
    before = c.pool.clone()
    into, outof = [2 * i for i in range(n)], [2 * i + 1 for i in range(n)]
    outof[298] = 2 * 17  # what sequence 17 reads
    c.prompt(into, outof)
    with pytest.raises(qe_moe.QeError, match="slot"):
        c.h.check()
    for i in (0, 4, 7, 17, 255, 256, 299):
        o, S = c.expect(i, before[2 * i])
        if lens[i]:
            c.close(c.out[c.cu[i]: c.cu[i + 1]], o, i)
            c.close(c.pool[2 * i + 1], S, i)
        else:
            assert torch.equal(c.pool[2 * i + 1], before[2 * i])
    assert bool((c.out[c.cu[298]: c.cu[299]] == 0).all()) and torch.equal(c.pool[34], before[34])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hk,hv", [(16, 32), (10, 30)])
def test_prompts_of_more_heads_and_chunks_than_run_at_once(hk, hv, dtype):
    """The matrices of a key head's value heads are made one after the other then."""
    c = Case(hk, hv, 64, 64, dtype, [1500, 300])
    w = [c.expect(i, c.pool[2 * i]) for i in range(2)]
    c.prompt([0, 2], [1, 3])
    c.h.check()
    for i in range(2):
        c.close(c.out[c.cu[i]: c.cu[i + 1]], w[i][0], i)
        c.close(c.pool[2 * i + 1], w[i][1], i)


def test_prompt_without_tokens_passes_states_on():
    c = Case(2, 4, 64, 128, torch.float16, [0, 0, 0])
    before = c.pool.clone()
    c.prompt([0, -1, 4], [1, 2, -1])
    c.h.check()
    assert torch.equal(c.pool[1], before[0]) and bool((c.pool[2] == 0).all())
    assert torch.equal(c.pool[[0, 3, 4, 5]], before[[0, 3, 4, 5]])


def test_states_near_the_end_of_the_range():
    """Nothing but the sequences' own tokens is computed from large states: no infinity out of a chunk's unused rows."""
    c = Case(1, 2, 64, 64, torch.float32, [1, 5, 70])
    c.pool.mul_(1e37)
    w = [c.expect(i, c.pool[2 * i]) for i in range(3)]
    c.prompt([0, 2, 4], [1, 3, 5])
    c.h.check()
    for i in range(3):
        c.close(c.out[c.cu[i]: c.cu[i + 1]], w[i][0], i)
        c.close(c.pool[2 * i + 1], w[i][1], i)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_prompt(dtype):
    c = Case(2, 4, 128, 128, dtype, [2000])
    o, S = c.expect(0, c.pool[0])
    c.prompt([0], [1])
    c.close(c.out, o)
    c.close(c.pool[1], S)


def test_a_prompt_is_its_tokens_one_by_one():
    """Chunked, recurrent, and in two parts: the same tokens leave the same state."""
    c = Case(2, 4, 128, 64, torch.float32, [150], slots=4)
    c.prompt([-1], [0])
    whole = c.out.clone()
    parts = torch.empty_like(whole)
    one = Case(2, 4, 128, 64, torch.float32, [1], slots=4)
    one.pool = c.pool
    for t in range(150):
        for name in ("q", "k", "v", "g", "beta"):
            setattr(one, name, getattr(c, name)[t: t + 1].contiguous())
        one.decode([1 if t else -1], [1], out=parts[t: t + 1])
    assert R.rel(parts, whole) <= TOL32 and R.rel(c.pool[1], c.pool[0]) <= TOL32
    c.prompt([-1], [2], cu=[0, 101])
    c.prompt([2], [2], cu=[101, 150])
    assert R.rel(c.out, whole) <= TOL32 and R.rel(c.pool[2], c.pool[0]) <= TOL32


@pytest.mark.parametrize("l2norm,scale", [(False, 0.0), (True, 0.7), (False, 0.01)])
def test_norm_and_scale(l2norm, scale):
    c = Case(2, 2, 64, 64, torch.float32, [100, 3])
    c.desc = dict(l2norm=l2norm, scale=scale)
    if not l2norm:
        c.k *= 0.2  # keys of length up to about one, as the rule needs them to be
    c.h = qe_mixer.GatedDelta(2, 2, 64, 64, t_max=103, seqs_max=103, **c.desc)
    for i in range(2):
        o, S = c.expect(i, c.pool[2 * i])
        c.prompt([0, 2], [1, 3])
        c.close(c.out[c.cu[i]: c.cu[i + 1]], o)
        c.close(c.pool[2 * i + 1], S)
    o, S = c.expect(1, c.pool[2])
    d = Case(2, 2, 64, 64, torch.float32, [1])
    d.pool = c.pool.clone()
    for name in ("q", "k", "v", "g", "beta"):
        setattr(d, name, getattr(c, name)[100:101].contiguous())
    d.h, d.desc = c.h, c.desc
    w, _ = d.expect(0, c.pool[2])
    d.decode([2], [3])
    d.close(d.out, w)


@pytest.mark.parametrize("rates", [(1e-6, 1e-5), (5.0, 50.0)])
def test_slow_and_fast_decay(rates):
    c = Case(2, 4, 128, 128, torch.float32, [400], rates=rates)
    o, S = c.expect(0, c.pool[0])
    c.prompt([0], [1])
    c.close(c.out, o)
    c.close(c.pool[1], S)


def test_a_state_that_is_cleared_within_a_prompt():
    """g of minus infinity, and very negative: nothing from before is left, and what follows keeps its 32 bits."""
    c = Case(2, 2, 64, 64, torch.float32, [130])
    c.g[20], c.g[70, 0], c.g[71, 1], c.g[100] = -math.inf, -3e38, -500.0, -20000.0
    o, S = c.expect(0, c.pool[0])
    c.prompt([0], [1])
    c.close(c.out, o)
    c.close(c.pool[1], S)
    d = Case(2, 2, 64, 64, torch.float32, [1])
    d.g[:] = -math.inf
    o, S = d.expect(0, d.pool[0])
    d.decode([0], [1])
    d.close(d.out, o)
    d.close(d.pool[1], S)


def test_zero_keys_and_gates():
    c = Case(2, 2, 64, 64, torch.float32, [70])
    c.q[5], c.k[7], c.beta[9], c.v[11] = 0, 0, 0, 0
    o, S = c.expect(0, c.pool[0])
    c.prompt([0], [1])
    c.close(c.out, o)
    c.close(c.pool[1], S)


def test_strided_rows_and_rows_of_no_sequence():
    c = Case(2, 4, 128, 64, torch.bfloat16, [30, 41])
    o = [c.expect(i, c.pool[2 * i]) for i in range(2)]
    T = c.T + 9
    wide = torch.full((T, 2 * 2 * 128 + 4 * 64 + 8), math.nan, dtype=torch.bfloat16, device="cuda")
    q, k, v = wide[:, :256], wide[:, 256:512], wide[:, 512:768]
    for a, b in ((q, c.q), (k, c.k), (v, c.v)):
        a[4: 4 + c.T] = b.reshape(c.T, -1)
    g, beta = (torch.full((T, 4), math.nan, device="cuda") for _ in range(2))
    g[4: 4 + c.T], beta[4: 4 + c.T] = c.g, c.beta
    out = torch.full((T, 4 * 64 + 16), 7.0, dtype=torch.bfloat16, device="cuda")
    h = qe_mixer.GatedDelta(2, 4, 128, 64, dtype=torch.bfloat16, t_max=T, seqs_max=2)
    h.prompt(q, k, v, g, beta, c.pool, ints([0, 2]), ints([1, 3]), ints([4, 34, 75]), out[:, :256])
    h.check()
    for i in range(2):
        c.close(out[4 + c.cu[i]: 4 + c.cu[i + 1], :256].reshape(-1, 4, 64), o[i][0])
        c.close(c.pool[2 * i + 1], o[i][1])
    assert bool((out[:4] == 7).all()) and bool((out[4 + c.T:] == 7).all()) and bool((out[:, 256:] == 7).all())


def test_slots_that_may_not_be_used():
    c = Case(1, 2, 64, 64, torch.float32, [20, 20, 20], slots=4)
    before = c.pool.clone()
    w = [[c.expect(i, before[s])[0] for s in range(4)] for i in range(3)]
    st = [[c.expect(i, before[s])[1] for s in range(4)] for i in range(3)]
    one = Case(1, 2, 64, 64, torch.float32, [1, 1, 1], slots=4)
    # slots in, slots out, which are computed, what is said
    for into, outof, fine, word in (
            ([0, 1, 2], [0, 3, 3], [1, 1, 0], "another"),     # the same slot written twice: the first writes it
            ([0, 1, 2], [1, 0, 3], [0, 0, 1], "another"),     # two states exchanged: each writes what the other reads
            ([0, 0, 0], [0, 1, 2], [0, 1, 1], "another"),     # one state continued three times, once over itself
            ([0, 0, 0], [3, 1, 2], [1, 1, 1], None),          # ... and kept
            ([0, 4, 1], [2, 3, 3], [1, 0, 0], "."),           # outside the pool
            ([0, -2, 1], [2, -1, 3], [1, 0, 1], "outside"),
            ([0, 1, 2], [3, 1, -5], [1, 1, 0], "outside")):
        for kind in ("prompt", "decode"):
            x = c if kind == "prompt" else one
            x.pool.copy_(before)
            x.out.fill_(7.0)
            getattr(x, kind)(into, outof)
            if word is None:
                x.h.check()
            else:
                with pytest.raises(qe_moe.QeError, match=word):
                    x.h.check()
            x.h.check()
            for i in range(3):
                rows = x.out[x.cu[i]: x.cu[i + 1]]
                if not fine[i]:
                    assert bool((rows == 0).all()), (into, outof, i, kind)
                else:
                    o, S = (w[i][into[i]], st[i][into[i]]) if kind == "prompt" else x.expect(i, before[into[i]])
                    x.close(rows, o)
                    if outof[i] >= 0:
                        x.close(x.pool[outof[i]], S)
            for s in set(range(4)) - {outof[i] for i in range(3) if fine[i]}:
                assert torch.equal(x.pool[s], before[s]), (into, outof, s, kind)


def test_bad_offsets_are_reported():
    c = Case(1, 1, 64, 64, torch.float32, [20, 20])
    for cu in ([0, 20, 1000], [0, 20, 10], [-5, 20, 40]):
        c.prompt([0, 2], [1, 3], cu=cu)
        with pytest.raises(qe_moe.QeError, match="offset"):
            c.h.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_offsets_outside_the_call_give_zeros_and_an_error(dtype):
    c = Case(2, 4, 64, 128, dtype, [70, 130, 50])
    before = c.pool.clone()
    w = [c.expect(i, before[2 * i]) for i in range(3)]
    for cu, fine, lost in (([-5, 70, 200, 250], [1, 2], [(0, 70)]), ([-(1 << 31), 70, 200, 250], [1, 2], [(0, 70)]),
                           ([0, 70, 200, 251], [0, 1], [(200, 250)]), ([0, 70, 1 << 30, (1 << 31) - 1], [0], [(70, 250)])):
        c.pool.copy_(before)
        c.out.fill_(7.0)
        c.prompt([0, 2, 4], [1, 3, 5], cu=cu)
        with pytest.raises(qe_moe.QeError, match="offset"):
            c.h.check()
        for a, b in lost:
            assert bool((c.out[a:b] == 0).all()), cu
        for i in range(3):
            if i in fine:
                c.close(c.out[c.cu[i]: c.cu[i + 1]], w[i][0], (cu, i))
                c.close(c.pool[2 * i + 1], w[i][1], (cu, i))
            else:
                assert torch.equal(c.pool[2 * i + 1], before[2 * i + 1]), (cu, i)


def test_refusals():
    c = Case(2, 4, 64, 64, torch.float32, [3, 4])
    a = dict(q=c.q, k=c.k, v=c.v, g=c.g, beta=c.beta, pool=c.pool, slots_in=ints([0, 2]), slots_out=ints([1, 3]), cu=ints(c.cu), out=c.out)
    for bad in (dict(q=c.q.half()), dict(k=c.k[:3]), dict(v=c.v.cpu()), dict(g=c.g.double()), dict(g=c.g.T.contiguous().T),
                dict(beta=c.beta[:, :2]), dict(pool=c.pool.half()), dict(pool=c.pool[:, :2]), dict(slots_in=ints([0])),
                dict(slots_out=ints([1, 3]).long()), dict(cu=ints([0, 3])), dict(out=c.out.bfloat16())):
        with pytest.raises(ValueError):
            c.h.prompt(**{**a, **bad})
    with pytest.raises(qe_moe.QeError, match="n_seqs"):
        c.h.prompt(**{**a, **dict(slots_in=ints([0, 1, 2]), slots_out=ints([3, 3, 3]), cu=ints([0, 1, 2, 3]))})
    small = qe_mixer.GatedDelta(2, 4, 64, 64, t_max=6, seqs_max=2)
    with pytest.raises(qe_moe.QeError, match="n_tokens"):
        small.prompt(**a)
    with pytest.raises(qe_moe.QeError, match="an input"):
        c.h.prompt(**{**a, **dict(out=c.v)})
    c.h.check()


def test_captured_steps_follow_the_slots_in_device_memory():
    """A prompt and a decode step in a graph, replayed on new inputs and slots with eager work between."""
    c = Case(2, 4, 128, 128, torch.bfloat16, [1, 1, 1], slots=8)
    p = Case(2, 4, 128, 128, torch.bfloat16, [70, 9], slots=8, seed=4)
    p.pool = c.pool
    into, outof, pin, pout, cu = ints([0, 1, 2]), ints([0, 1, 2]), ints([-1, 3]), ints([4, 3]), ints(p.cu)

    def calls(stream, out, pool, pout_):
        c.h.decode(c.q, c.k, c.v, c.g, c.beta, pool, into, outof, out, stream=stream)
        p.h.prompt(p.q, p.k, p.v, p.g, p.beta, pool, pin, pout, cu, pout_, stream=stream)

    mine, o1, o2 = c.pool.clone(), torch.empty_like(c.out), torch.empty_like(p.out)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        calls(side, o1, mine.clone(), o2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(torch.cuda.current_stream(), o1, mine, o2)
    g = gen(9)
    for step in range(4):
        c.v.copy_(torch.randn(c.v.shape, generator=g, device="cuda"))
        into.copy_(ints([step, step + 1, 7])), outof.copy_(ints([step, step + 1, 7]))
        pin.copy_(ints([-1, 6])), pout.copy_(ints([6 - step % 2, 6])) if step % 2 else pout.copy_(ints([-1, 6]))
        if step == 3:
            into.copy_(ints([0, 1, 2])), outof.copy_(ints([0, 1, 2]))
        graph.replay()
        torch.cuda.synchronize()
        e1, e2 = torch.empty_like(o1), torch.empty_like(o2)
        calls(None, e1, c.pool, e2)
        torch.cuda.synchronize()
        assert torch.equal(o1, e1) and torch.equal(o2, e2) and torch.equal(mine, c.pool), step
    c.h.check(), p.h.check()


@pytest.mark.parametrize("l2norm", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_keys_and_queries_whose_squares_pass_32_bits_are_not_finite(dtype, l2norm):
    """In prompts and single steps alike: from the token on for a key, the token's own outputs for a query."""
    c, one = Case(1, 2, 64, 64, dtype, [40, 30]), Case(1, 2, 64, 64, dtype, [1, 1])
    for x in (c, one):
        x.h = qe_mixer.GatedDelta(1, 2, 64, 64, dtype=dtype, t_max=70, seqs_max=2, l2norm=l2norm)
        if not l2norm:
            x.k *= 0.2
    for x, kind, at in ((c, "prompt", 20), (one, "decode", 0)):
        getattr(x, kind)([0, 2], [1, 3])
        clean, pool, end = x.out.clone(), x.pool.clone(), x.cu[1]
        assert bool(torch.isfinite(clean).all())
        keep = x.k.clone()
        x.k[at, 0, 5] = 3e19
        getattr(x, kind)([0, 2], [1, 3])
        x.k.copy_(keep)
        assert bool(x.out[at:end].isnan().all()) and bool(x.pool[1].isnan().all()), kind
        assert torch.equal(x.out[:at], clean[:at]) and torch.equal(x.out[end:], clean[end:]) and torch.equal(x.pool[3], pool[3])
        if l2norm:
            x.q[at, 0, 5] = 3e19
            getattr(x, kind)([0, 2], [1, 3])
            assert bool(x.out[at].isnan().all()), kind
            assert torch.equal(x.out[:at], clean[:at]) and torch.equal(x.out[at + 1:], clean[at + 1:]) and torch.equal(x.pool[1], pool[1])
        x.h.check()


@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_that_are_not_finite_reach_no_earlier_token(what, dtype):
    c = Case(1, 2, 64, 64, dtype, [100, 40])
    c.prompt([0, 2], [1, 3])
    clean, pool = c.out.clone(), c.pool.clone()
    for name in ("q", "k", "v", "g", "beta"):
        x = getattr(c, name)
        if name == "g" and what == math.inf:
            continue
        keep = x.clone()
        x.select(0, 71).view(-1)[0] = what
        c.prompt([0, 2], [1, 3])
        setattr(c, name, keep)
        assert torch.equal(c.out[:71], clean[:71]), name
        assert torch.equal(c.out[100:], clean[100:]) and torch.equal(c.pool[3], pool[3]), name
        assert not bool(torch.isfinite(c.out[71]).all()), name
        if name == "v":  # one column of one head
            assert torch.equal(c.out[:, 1], clean[:, 1]) and torch.equal(c.out[:, 0, 1:], clean[:, 0, 1:])
            assert not bool(torch.isfinite(c.out[71:100, 0, 0]).any()) and not bool(torch.isfinite(c.pool[1, 0, :, 0]).any())
