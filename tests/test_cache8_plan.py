"""How calls over an 8-bit cache, and of sequences that share their beginnings, are cut up (CPU)."""
import ctypes
import itertools
import os
import subprocess

import numpy as np
import pytest

from conftest import PKG

SHIM = """
#include "qe_mixer_plan.h"
extern "C" {
void decode8_plan(long seqs, long heads, long len, int *steps, int *splits) { qe_attn_decode8_plan(seqs, heads, len, steps, splits); }
int decode_steps(int len, int steps, int splits) { return qe_attn_decode_steps(len, steps, splits); }
int decode_active(int len, int steps) { return qe_attn_decode_active(len, steps); }
int prompt8_halves(long tiles, int bn, long len) { return qe_attn_prompt8_halves(tiles, bn, len); }
void prompt8_plan(long tiles, int bm, int bn, long len, int *steps, int *splits) { qe_attn_prompt8_plan(tiles, bm, bn, len, steps, splits); }
int tile_steps(int len, int b, int e, int r, int g, int bm, int bn) { return qe_attn_tile_steps(len, b, e, r, g, bm, bn); }
int tile_splits(int n, int steps, int splits) { return qe_attn_tile_splits(n, steps, splits); }
void split_range(int n, int splits, int s, int *lo, int *hi) { qe_split_range(n, splits, s, lo, hi); }
int prompt_rows(int n, int s, int g, int h, int d) { return qe_attn_prompt_rows(n, s, g, h, d); }
int max_tiles(int n, int s, int g, int bm) { return qe_attn_max_tiles(n, s, g, bm); }
int shared_seqs(int n, int h) { return qe_attn_shared_seqs(n, h); }
void shared_plan(int n, int q, int kv, long prefix, long own, int *p, int *steps, int *splits) { qe_attn_shared_plan(n, q, kv, prefix, own, p, steps, splits); }
int shared_per(int n, int step, int p) { return qe_attn_shared_per(n, step, p); }
int shared_active(int n, int step, int p) { return qe_attn_shared_active(n, step, p); }
int shared_rows() { return QE_ATTN_SHARED_ROWS; }
int prompt8_rows() { return QE_ATTN_PROMPT8_ROWS; }
int part_wgs() { return QE_ATTN_PART_WGS; }
int decode_splits() { return QE_ATTN_DECODE_SPLITS; }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("cache8_plan")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-shared", "-fPIC", "-std=c++17", "-Wall", "-Wno-unused-function", "-I", os.path.join(PKG, "csrc"),
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    lib = ctypes.CDLL(str(d / "shim.so"))
    lib.decode8_plan.argtypes = [ctypes.c_long] * 3 + [ctypes.c_void_p] * 2
    lib.prompt8_halves.argtypes = [ctypes.c_long, ctypes.c_int, ctypes.c_long]
    lib.prompt8_plan.argtypes = [ctypes.c_long, ctypes.c_int, ctypes.c_int, ctypes.c_long, ctypes.c_void_p, ctypes.c_void_p]
    lib.shared_plan.argtypes = [ctypes.c_int] * 3 + [ctypes.c_long] * 2 + [ctypes.c_void_p] * 3
    return lib


def ints(n):
    x = [ctypes.c_int() for _ in range(n)]
    return x, [ctypes.byref(i) for i in x]


LENS = (1, 16, 33, 700, 5000, 8111, 60000, 1 << 20, 1 << 30)


def test_decode8_workgroups_cover_every_length(plan):
    for seqs, heads, longest in itertools.product((1, 2, 9, 24, 300, 65535), (1, 2, 8, 256), LENS):
        (steps, splits), refs = ints(2)
        plan.decode8_plan(seqs, heads, longest, *refs)
        steps, splits = steps.value, splits.value
        assert steps >= 2 and 1 <= splits <= plan.decode_splits()
        if splits > 1:  # partial results have room
            assert seqs * heads * splits <= plan.part_wgs()
        for n in {1, 31, 32, longest // 3 + 1, longest, min(1 << 30, 2 * longest)}:  # the host may have believed less
            mine = plan.decode_steps(n, steps, splits)
            active = plan.decode_active(n, mine)
            assert active <= splits and (active - 1) * mine < -(-n // 32) <= active * mine


def test_prompt8_splits_fit_their_scratch_and_cover_a_tiles_steps(plan):
    rng = np.random.default_rng(0)
    for _ in range(3000):
        n, seqs = int(np.exp(rng.uniform(0, np.log(60000)))), int(rng.integers(1, 40))
        group, heads, dim = int(rng.choice([1, 4, 7, 8, 16])), int(rng.choice([1, 2, 8, 64])), int(rng.choice([64, 128, 256]))
        bm, bn = plan.prompt_rows(n, seqs, group, heads, dim), 32 if dim == 256 else 64
        tiles = plan.max_tiles(n, seqs, group, bm) * heads
        longest = int(np.exp(rng.uniform(0, np.log(1 << 30))))
        (steps, splits), refs = ints(2)
        plan.prompt8_plan(tiles, bm, bn, longest, *refs)
        steps, splits = steps.value, splits.value
        assert steps >= 8 and splits >= 1
        assert splits == 1 or tiles * splits * bm <= plan.prompt8_rows()
        if plan.prompt8_halves(tiles, bn, longest):  # eight waves join in LDS, and have all of a tile's steps
            assert splits == 1 and dim < 256 and bm == 128 and 128 < tiles <= 512
        for own in (0, 1, 7, 8, 9, steps, steps + 1, int(rng.integers(0, 3 * steps * splits + 2))):
            mine = plan.tile_splits(own, steps, splits)
            assert 1 <= mine <= splits and (mine == 1) == (own <= steps or splits == 1)
            at = 0
            for s in range(mine):
                (lo, hi), refs = ints(2)
                plan.split_range(own, mine, s, *refs)
                assert lo.value == at
                at = hi.value
            assert at == own


def test_a_tiles_steps_end_at_its_last_rows_position(plan):
    for group, bm, bn in itertools.product((1, 3, 8), (128, 256), (32, 64)):
        for tokens, length in ((1, 1), (5, 3), (100, 100), (300, 5000), (40, 0), (700, 20)):
            rows = tokens * group
            for row0 in range(0, rows, bm):
                last = length - tokens + (min(row0 + bm, rows) - 1) // group  # place of the last row
                assert plan.tile_steps(length, 10, 10 + tokens, row0, group, bm, bn) == max(0, -(-(last + 1) // bn))


def test_shared_partial_results_fit_their_scratch(plan):
    rng = np.random.default_rng(1)
    for _ in range(4000):
        heads, group = int(rng.choice([1, 2, 8, 40, 256])), int(rng.integers(1, 17))
        seqs = int(np.exp(rng.uniform(0, np.log(65535))))
        n = plan.shared_seqs(seqs, heads * group)
        assert 8 <= n <= seqs or n == seqs
        prefix, own = (int(np.exp(rng.uniform(0, np.log(1 << 30)))) for _ in range(2))
        (p, steps, splits), refs = ints(3)
        plan.shared_plan(n, heads * group, heads, prefix, own, *refs)
        assert p.value >= 1 and splits.value >= 1 and n * heads * group * (p.value + splits.value) <= plan.shared_rows()


def test_shared_splits_cover_every_prefix(plan):
    for step, p in itertools.product((32, 64), (1, 2, 7, 32, 250)):
        for n in (0, 1, 31, 32, 33, 64, 65, 1000, 16000, 1 << 30):
            per, active = plan.shared_per(n, step, p), plan.shared_active(n, step, p)
            steps = -(-n // step)
            assert active <= p and active * per >= steps and (active == 0 or (active - 1) * per < steps)
