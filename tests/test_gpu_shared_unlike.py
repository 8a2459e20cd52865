"""Sequences that share their beginnings, whose own positions the hints say nothing of: as test_gpu_shared.py."""
import pytest

torch = pytest.importorskip("torch")
from test_gpu_shared import CACHES, Grouped, close  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("heads", [(16, 2, 256, 256), (32, 8, 128, 64), (3, 3, 64, 16)])
@pytest.mark.parametrize("groups,own,prefix,before,behind", [
    ([4], [10, 3, 1, 0, 6000], [3000], 0, 1),  # a long one of no group behind
    ([3, 2], [5000, 2, 1, 0, 2500, 33], [4000, 70], 1, 0),  # one before, and one behind a short prefix
    ([2] * 9, [40 + i for i in range(18)], [500 + 77 * i for i in range(9)], 0, 0)])  # many small groups
def test_own_parts_of_all_lengths(heads, groups, own, prefix, before, behind, cache):
    g = Grouped(heads, torch.bfloat16, cache, groups, own, prefix, before=before, behind=behind)
    q = g.c.q(len(own))
    want, off = g.expect(q)
    for hints in ((0, 0), (max(g.c.kv_len), max(prefix)), (0, max(prefix)), (max(g.c.kv_len), 0), (max(g.c.kv_len), max(g.c.kv_len)), (1, 1)):
        out, again = torch.full_like(q, 7.0), torch.empty_like(q)
        g.run(q, out, *hints)
        g.run(q, again, *hints)
        g.c.att.check()
        close(out, want, off)
        assert torch.equal(out, again)


@pytest.mark.parametrize("cache", CACHES)
def test_wide_tables(cache):
    """Room for far more positions than there are, without a hint: prefixes on either side of what is assumed."""
    for groups, own, prefix in (([3, 2], [400, 2, 0, 33, 1], [700, 5]), ([2], [10, 300], [20000])):
        g = Grouped((8, 2, 128, 64), torch.float16, cache, groups, own, prefix, behind=0)
        n = len(own)
        table = torch.full((n, 262144 // 64), 1 << 30, dtype=torch.int32, device="cuda")
        table[:, : g.c.table.shape[1]] = g.c.table
        q = g.c.q(n)
        out = torch.full_like(q, 7.0)
        g.run(q, out, table=table)
        g.c.att.check()
        close(out, *g.expect(q))
