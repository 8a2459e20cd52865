"""The tests' own idea of when eight waves share a prompt's tile, against the plan's (CPU)."""
import types

import numpy as np
import pytest

pytest.importorskip("torch")
from test_cache8_plan import plan  # noqa: E402, F401
from test_gpu_attention8 import in_halves  # noqa: E402


def test_in_halves_is_as_planned(plan):  # noqa: F811
    rng = np.random.default_rng(3)
    seen = set()
    for _ in range(5000):
        group, hkv, n = int(rng.choice([1, 3, 4, 7])), int(rng.choice([1, 2, 8, 12])), int(rng.integers(1, 9))
        tokens, longest = int(np.exp(rng.uniform(0, np.log(9000)))), int(np.exp(rng.uniform(0, np.log(9000))))
        c = types.SimpleNamespace(hq=group * hkv, hkv=hkv)
        want = bool(plan.prompt8_halves(plan.max_tiles(tokens, n, group, 128) * hkv, 64, longest))
        # (from 64 steps on the plan takes splits; the tests' calls have fewer)
        if longest <= 63 * 64:
            assert bool(in_halves(c, tokens, n, longest)) == want, (group, hkv, n, tokens, longest)
            seen.add(want)
    assert seen == {True, False}
