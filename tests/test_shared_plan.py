"""How calls of sequences that share their beginnings are cut up where the host's hints say little of a sequence's own positions (CPU)."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from conftest import PKG

SHIM = """
#include "qe_mixer_plan.h"
extern "C" {
int shared_seqs(int n, int h) { return qe_attn_shared_seqs(n, h); }
void shared_plan(int n, int q, int kv, long prefix, long own, int *p, int *steps, int *splits, long len) {
    qe_attn_shared_plan(n, q, kv, prefix, own, p, steps, splits, len);
}
int shared_rows() { return QE_ATTN_SHARED_ROWS; }
int decode_steps(int len, int steps, int splits) { return qe_attn_decode_steps(len, steps, splits); }
int decode_active(int len, int steps) { return qe_attn_decode_active(len, steps); }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("shared_plan")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-shared", "-fPIC", "-std=c++17", "-Wall", "-Wno-unused-function", "-I", os.path.join(PKG, "csrc"),
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    lib = ctypes.CDLL(str(d / "shim.so"))
    lib.shared_plan.argtypes = [ctypes.c_int] * 3 + [ctypes.c_long] * 2 + [ctypes.c_void_p] * 3 + [ctypes.c_long]

    def of(n, q, kv, max_len, max_prefix, table=None):
        """As a call with these hints is planned, 0: not stated, whose table has room for `table` positions.  -> prefix splits, steps,
        splits"""
        p, steps, splits = (ctypes.c_int() for _ in range(3))
        own = max(1, max_len - max_prefix) if max_len and max_prefix else 0
        max_len = max_len or table
        lib.shared_plan(n, q, kv, min(max_prefix or 16384, max_len), own, *(ctypes.byref(x) for x in (p, steps, splits)), max_len)
        return p.value, steps.value, splits.value

    lib.of = of
    return lib


def longest_share(plan, own, steps, splits):
    """Steps of 32 keys that one workgroup has of `own` positions."""
    return min(plan.decode_steps(own, steps, splits), -(-own // 32))


def test_own_positions_without_a_hint_are_split(plan):
    """32 sequences of 16 / 2 heads with up to 1500 of their own behind 8000: 47 steps in a row of one workgroup would be as long as the call."""
    for max_len, table in ((9501, 9504), (0, 9504), (0, 1 << 20), (0, 1 << 30)):
        for max_prefix in (0, 8000):
            _, steps, splits = plan.of(32, 16, 2, max_len, max_prefix, table)
            assert longest_share(plan, 1501, steps, splits) <= 8, (max_len, table, max_prefix, steps, splits)
    _, steps, splits = plan.of(32, 16, 2, 9501, 8000)  # exact hints: twelve workgroups for the longest
    assert plan.decode_active(1501, plan.decode_steps(1501, steps, splits)) == 12


def test_own_positions_that_the_hints_do_not_bound_are_split(plan):
    """A long sequence of no group, or of a group with a short prefix, beside a long prefix."""
    for n, q, kv, max_len, max_prefix, own in ((9, 16, 2, 30010, 30000, 30000), (8, 16, 2, 60000, 59900, 60000), (14, 16, 2, 16010, 16000, 2000), (14, 16, 2, 16010, 0, 2000)):
        _, steps, splits = plan.of(n, q, kv, max_len, max_prefix)
        # of the 1024 workgroups it has its share, of at least eight steps
        share = 1024 // (n * kv)
        assert longest_share(plan, own, steps, splits) <= max(8, -(-(-(-own // 32)) // share)), (n, steps, splits)


def test_partial_results_fit_and_cover(plan):
    rng = np.random.default_rng(7)
    for _ in range(4000):
        heads, group = int(rng.choice([1, 2, 8, 40, 256])), int(rng.integers(1, 17))
        seqs = int(np.exp(rng.uniform(0, np.log(65535))))
        n = plan.shared_seqs(seqs, heads * group)
        max_len = int(np.exp(rng.uniform(0, np.log(1 << 30))))
        max_prefix = int(rng.choice([0, 1, max_len // 2, max_len]))
        p, steps, splits = plan.of(n, heads * group, heads, int(rng.choice([0, max_len])), max_prefix, max_len)
        assert p >= 1 and splits >= 1 and steps >= 2 and n * heads * group * (p + splits) <= plan.shared_rows()
        assert n * heads * splits <= max(2048 + n * heads, 1024)
        for own in (1, 31, 33, max_len):
            mine = plan.decode_steps(own, steps, splits)
            active = plan.decode_active(own, mine)
            assert active <= splits and (active - 1) * mine < -(-own // 32) <= active * mine
