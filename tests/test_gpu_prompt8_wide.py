"""Prompts over an 8-bit cache whose tables have room for far more than they hold, without a word of their lengths."""
import pytest

torch = pytest.importorskip("torch")
import cache8_ref as Q  # noqa: E402
import qe_mixer  # noqa: E402
import qe_moe  # noqa: E402
from cache8_ref import Case8, ints  # noqa: E402
from test_gpu_attention8 import close, offsets  # noqa: E402

pytestmark = pytest.mark.gpu
CASES = [(32, 8, 128, 16, [300, 500, 100], [0, 0, 6000]),  # eight waves in halves, and splits of some of their tiles
         (24, 8, 64, 32, [700, 64, 33], [0, 9000, 40]),
         (16, 2, 256, 64, [30, 5, 1], [7000, 100, 2999]), (16, 2, 256, 64, [1000, 40], [0, 5000]), (32, 16, 256, 32, [900, 333], [100, 4000]),
         (8, 2, 128, 16, [200, 0, 9], [3000, 5, 0]), (4, 4, 64, 16, [1], [0])]


@pytest.mark.parametrize("dtype,codes", [(torch.bfloat16, torch.int8), (torch.float16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("hq,hkv,dim,page,lens,ctx", CASES)
def test_wide_tables(hq, hkv, dim, page, lens, ctx, dtype, codes):
    c = Case8(hq, hkv, dim, page, dtype, codes, [a + b for a, b in zip(lens, ctx)], extra_cols=262144 // page)
    cu = offsets(lens)
    q = c.q(cu[-1] + 2)
    want, off = Q.attend_batch(c, q[: cu[-1]], cu)
    out, again = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    c.att.prompt8(c.batch(cu), q, c.cache(), out)
    c.att.prompt8(c.batch(cu), q, c.cache(), again)
    c.att.check()
    close(out[: cu[-1]], want, off)
    assert bool((out[cu[-1]:] == 7).all()) and torch.equal(out, again)


@pytest.mark.parametrize("hq,hkv,dim,page,lens,ctx", CASES[:4])
def test_bad_pages_and_lengths(hq, hkv, dim, page, lens, ctx):
    c = Case8(hq, hkv, dim, page, torch.bfloat16, torch.int8, [a + b for a, b in zip(lens, ctx)], extra_cols=262144 // page)
    cu = offsets(lens)
    q = c.q(cu[-1])
    want, off = Q.attend_batch(c, q, cu)
    for i in range(len(lens)):
        for page_of, kv in ((0, None), ((c.kv_len[i] - 1) // page, None), (None, -1), (None, 1 << 30)):
            table, lengths = c.table.clone(), list(c.kv_len)
            if kv is None:
                table[i, page_of] = c.kc.shape[0]
            else:
                lengths[i] = kv
            out = torch.full_like(q, 7.0)
            c.att.prompt8(qe_mixer.Batch(ints(lengths), table, ints(cu)), q, c.cache(), out)
            with pytest.raises(qe_moe.QeError, match="page" if kv is None else "length"):
                c.att.check()
            rest = torch.ones(cu[-1], dtype=torch.bool, device="cuda")
            rest[cu[i]: cu[i + 1]] = False
            assert bool((out[~rest] == 0).all())
            close(out[rest], want[rest], off[rest])


def test_captured_lengths_grow():
    """The same call replayed while a sequence grows far beyond the call's tokens."""
    c = Case8(32, 8, 128, 16, torch.float16, torch.int8, [9000, 400], extra_cols=262144 // 16)
    q = c.q(900)
    kv, cu = ints([500, 400]), ints([0, 500, 900])
    b = qe_mixer.Batch(kv, c.table, cu)
    out = torch.empty_like(q)
    c.att.prompt8(b, q, c.cache(), out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.att.prompt8(b, q, c.cache(), out, stream=torch.cuda.current_stream())
    for n in (500, 9000, 2600, 700):
        c.kv_len = [n, 400]
        kv.copy_(ints(c.kv_len))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        close(out, *Q.attend_batch(c, q, [0, 500, 900]))
        eager = torch.empty_like(out)
        c.att.prompt8(b, q, c.cache(), eager)
        assert torch.equal(eager, out)
    c.att.check()
