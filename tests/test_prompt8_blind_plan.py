"""How prompts over an 8-bit cache are cut up where the host says nothing of their lengths (CPU)."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from conftest import PKG

SHIM = """
#include "qe_mixer_plan.h"
extern "C" {
int blind(long tiles, int bm, int bn, long tokens, long len, int *steps, int *splits) { return qe_attn_prompt8_blind(tiles, bm, bn, tokens, len, steps, splits); }
int prompt_rows(int n, int s, int g, int h, int d) { return qe_attn_prompt_rows(n, s, g, h, d); }
int max_tiles(int n, int s, int g, int bm) { return qe_attn_max_tiles(n, s, g, bm); }
int tile_splits(int n, int steps, int splits) { return qe_attn_tile_splits(n, steps, splits); }
int rows() { return QE_ATTN_PROMPT8_ROWS; }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("prompt8_blind")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-shared", "-fPIC", "-std=c++17", "-Wall", "-Wno-unused-function", "-I", os.path.join(PKG, "csrc"),
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    lib = ctypes.CDLL(str(d / "shim.so"))
    lib.blind.argtypes = [ctypes.c_long, ctypes.c_int, ctypes.c_int, ctypes.c_long, ctypes.c_long, ctypes.c_void_p, ctypes.c_void_p]

    def of(tokens, seqs, group, heads, dim, table):
        bm, bn = lib.prompt_rows(tokens, seqs, group, heads, dim), 32 if dim == 256 else 64
        tiles = lib.max_tiles(tokens, seqs, group, bm) * heads
        steps, splits = ctypes.c_int(), ctypes.c_int()
        halves = lib.blind(tiles, bm, bn, tokens, table, ctypes.byref(steps), ctypes.byref(splits))
        return bm, bn, tiles, bool(halves), steps.value, splits.value

    lib.of = of
    return lib


@pytest.mark.parametrize("table", [2048, 32768, 1 << 18, 1 << 30])
def test_a_wide_table_changes_little(plan, table):
    # new prompts: eight waves where their tiles are few, and no split of tiles that have no more steps than a fresh prompt's
    _, bn, _, halves, steps, splits = plan.of(900, 1, 4, 8, 128, table)
    assert halves and plan.tile_splits(-(-900 // bn), steps, splits) == 1
    _, bn, _, _, steps, splits = plan.of(8000, 1, 4, 8, 128, max(table, 8000))
    assert splits == 1
    # few tokens after many: split
    _, bn, tiles, _, steps, splits = plan.of(30, 1, 8, 2, 256, table)
    assert plan.tile_splits(2000 // bn, steps, splits) >= 4
    if table >= 32768:
        assert plan.tile_splits(10000 // bn, steps, splits) * tiles >= 128
        _, bn, tiles, _, steps, splits = plan.of(600, 1, 4, 8, 128, table)
        assert plan.tile_splits(20600 // bn, steps, splits) * tiles >= 512


def test_splits_fit_their_scratch(plan):
    rng = np.random.default_rng(5)
    for _ in range(5000):
        tokens, table = (int(np.exp(rng.uniform(0, np.log(x)))) for x in (60000, 1 << 30))
        bm, bn, tiles, halves, steps, splits = plan.of(tokens, int(rng.integers(1, 100)), int(rng.choice([1, 4, 7, 8, 16])), int(rng.choice([1, 2, 8, 64])),
                                                       int(rng.choice([64, 128, 256])), table)
        assert steps >= 8 and splits >= 1 and (splits == 1 or tiles * splits * bm <= plan.rows())
        assert splits == 1 or tiles * splits <= 1024
        assert not halves or (bm == 128 and bn == 64)
