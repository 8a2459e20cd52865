"""How calls of the token mixers are cut up, and which values from device memory are used (CPU)."""
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
void decode_plan(long seqs, long heads, int dim, long len, int *steps, int *splits) { qe_attn_decode_plan(seqs, heads, dim, len, steps, splits); }
int decode_steps(int len, int steps, int splits) { return qe_attn_decode_steps(len, steps, splits); }
int decode_active(int len, int steps) { return qe_attn_decode_active(len, steps); }
int prompt_splits(long tiles, long len) { return qe_attn_prompt_splits(tiles, len); }
int first_tile(int cu, int i, int g, int bm) { return qe_attn_first_tile(cu, i, g, bm); }
int max_tiles(int n, int s, int g, int bm) { return qe_attn_max_tiles(n, s, g, bm); }
int first_chunk(int cu, int i) { return qe_delta_first_chunk(cu, i); }
int max_chunks(int n, int s) { return qe_delta_max_chunks(n, s); }
void split_range(int n, int splits, int s, int *lo, int *hi) { qe_split_range(n, splits, s, lo, hi); }
int checked(int v, int lo, int hi, int other, unsigned *bad) { return qe_checked(v, lo, hi, other, bad); }
int slot_pair(long n, int a, int b) { return qe_slot_pair(n, a, b); }
int slot_conflict(int i, int oi, int j, int ij, int oj) { return qe_slot_conflict(i, oi, j, ij, oj); }
int decode_once(long s, long h, int d, long n) { return qe_attn_decode_once(s, h, d, n); }
int fits(long wgs, int threads) { return qe_fits_launch(wgs, threads); }
void rows_of(int a, int b, int n, int *lo, int *hi, unsigned *bad) { qe_rows_of(a, b, n, lo, hi, bad); }
int bad_offsets(int a, int b, int n) { return qe_bad_offsets(a, b, n); }
int wgs() { return QE_ATTN_WGS; }
int decode_wgs() { return QE_ATTN_DECODE_WGS; }
int decode_splits() { return QE_ATTN_DECODE_SPLITS; }
int part_wgs() { return QE_ATTN_PART_WGS; }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("mixer_plan")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-shared", "-fPIC", "-std=c++17", "-Wall", "-Wno-unused-function", "-I", os.path.join(PKG, "csrc"),
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    lib = ctypes.CDLL(str(d / "shim.so"))
    lib.prompt_splits.argtypes = [ctypes.c_long, ctypes.c_long]
    lib.decode_plan.argtypes = [ctypes.c_long, ctypes.c_long, ctypes.c_int, ctypes.c_long, ctypes.c_void_p, ctypes.c_void_p]
    lib.decode_once.argtypes = [ctypes.c_long, ctypes.c_long, ctypes.c_int, ctypes.c_long]
    lib.fits.argtypes = [ctypes.c_long, ctypes.c_int]
    lib.slot_pair.argtypes = [ctypes.c_long, ctypes.c_int, ctypes.c_int]
    return lib


def decode_plan(plan, seqs, heads, dim, n):
    steps, splits = ctypes.c_int(), ctypes.c_int()
    plan.decode_plan(seqs, heads, dim, n, ctypes.byref(steps), ctypes.byref(splits))
    return steps.value, splits.value


def test_decode_workgroups_cover_every_length(plan):
    """Whatever the host believed the longest to be: all steps of 32 keys are some launched workgroup's, once."""
    for seqs, heads, dim in itertools.product((1, 2, 7, 24, 300, 65535), (1, 2, 8, 12, 256), (64, 256)):
        for told in (1, 31, 700, 8111, 100000, (1 << 31) - 1):
            steps, splits = decode_plan(plan, seqs, heads, dim, told)
            for n in (0, 1, 32, 33, 64, 65, 700, 8111, 100000, (1 << 31) - 32):
                tiles = -(-n // 32)
                mine = plan.decode_steps(n, steps, splits)
                active = plan.decode_active(n, mine)
                assert mine >= steps and active <= splits and active * mine >= tiles and (active - 1) * mine < max(tiles, 1)
                if n <= told:
                    assert mine == steps


def test_launches_have_less_than_2_32_threads(plan):
    for threads in (256, 512, 1024):
        for n in (1, 1 << 20, (1 << 32) // threads - 1, (1 << 32) // threads, (1 << 32) // threads + 1, 1 << 40):
            assert plan.fits(n, threads) == (n * threads < 1 << 32)


def test_large_calls_pass_the_caches_by(plan):
    for seqs, heads, dim in itertools.product((1, 2, 7, 24, 65535), (1, 8, 256), (64, 128, 256)):
        for n in (0, 1, 700, 8192, 100000, 1 << 30):
            size = seqs * heads * dim * 4 * n  # of the keys and values, two bytes each
            if size >= 32 << 20:
                assert plan.decode_once(seqs, heads, dim, n)
            elif size < 16 << 20 and seqs * heads * dim * 4 < 32 << 20:
                assert not plan.decode_once(seqs, heads, dim, n)


def test_partial_results_fit_their_scratch(plan):
    lens = [0, 1, 127, 128, 129, 1000, 65536, (1 << 31) - 1]
    for seqs, heads, dim in itertools.product([*range(1, 300), 2047, 2048, 65535], (1, 2, 3, 8, 256), (64, 256)):
        for n in lens:
            steps, s = decode_plan(plan, seqs, heads, dim, n)
            assert 1 <= s <= plan.decode_splits() and steps >= 2
            assert s == 1 or (seqs * heads < plan.decode_wgs() and seqs * heads * s <= plan.part_wgs())
    for tiles in list(range(1, 1200)) + [1 << 28]:
        for n in lens:
            s = plan.prompt_splits(tiles, n)
            assert s >= 1 and (s == 1 or tiles * s <= plan.wgs())


def test_split_ranges_cover_once(plan):
    lo, hi = ctypes.c_int(), ctypes.c_int()
    for n in (0, 1, 2, 3, 7, 64, 1000):
        for splits in (1, 2, 3, 5, 8, 100):
            seen = []
            for s in range(splits):
                plan.split_range(n, splits, s, ctypes.byref(lo), ctypes.byref(hi))
                assert 0 <= lo.value <= hi.value <= n
                seen += range(lo.value, hi.value)
            assert seen == list(range(n))


@pytest.mark.parametrize("group,bm", [(1, 128), (3, 128), (8, 128), (16, 128), (7, 256)])
def test_tiles_of_any_lengths_fit_and_do_not_meet(plan, group, bm):
    rng = np.random.default_rng(group)
    for _ in range(200):
        n = int(rng.integers(1, 9))
        lens = rng.integers(0, 300, n) * rng.integers(0, 2, n)
        cu = np.concatenate([[0], np.cumsum(lens)]) + int(rng.integers(0, 5))
        total = plan.max_tiles(int(cu[-1]), n, group, bm)
        end = 0
        for i in range(n):
            first = plan.first_tile(int(cu[i]), i, group, bm)
            assert first >= end
            end = first + -(-int(lens[i]) * group // bm)
        assert end <= total


def test_chunks_of_any_lengths_fit_and_do_not_meet(plan):
    rng = np.random.default_rng(1)
    for _ in range(200):
        n = int(rng.integers(1, 9))
        lens = rng.integers(0, 300, n) * rng.integers(0, 2, n)
        cu = np.concatenate([[0], np.cumsum(lens)]) + int(rng.integers(0, 70))
        end = 0
        for i in range(n):
            assert plan.first_chunk(int(cu[i]), i) >= end
            end = plan.first_chunk(int(cu[i]), i) + -(-int(lens[i]) // 64)
        assert end <= plan.max_chunks(int(cu[-1]), n)


def test_values_out_of_range_are_replaced_and_noted(plan):
    bad = ctypes.c_uint(0)
    assert plan.checked(5, 0, 5, 9, ctypes.byref(bad)) == 5 and plan.checked(0, 0, 5, 9, ctypes.byref(bad)) == 0 and bad.value == 0
    for v in (-1, 6, -(1 << 31), (1 << 31) - 1):
        bad.value = 0
        assert plan.checked(v, 0, 5, 3, ctypes.byref(bad)) == 3 and bad.value == 1


def test_offsets_that_are_none_are_found(plan):
    for a, b in ((0, 0), (0, 9), (9, 9), (3, 4)):
        assert not plan.bad_offsets(a, b, 9)
    for a, b in ((-1, 0), (-1, -1), (4, 3), (0, 10), (10, 10), (10, 9), (0, -1), (-(1 << 31), (1 << 31) - 1), ((1 << 31) - 1, -(1 << 31))):
        assert plan.bad_offsets(a, b, 9)


def test_rows_of_any_offsets_are_the_calls(plan):
    far = (-(1 << 31), -5, -1, 0, 1, 8, 9, 10, (1 << 31) - 1)
    lo, hi, bad = ctypes.c_int(), ctypes.c_int(), ctypes.c_uint()
    for a, b, n in itertools.product(far, far, (0, 1, 9)):
        bad.value = 0
        plan.rows_of(a, b, n, ctypes.byref(lo), ctypes.byref(hi), ctypes.byref(bad))
        assert 0 <= lo.value <= hi.value <= n
        assert set(range(lo.value, hi.value)) == {t for t in range(n) if a <= t < b}
        assert bad.value == (not 0 <= a <= b <= n)


def test_sequences_that_are_computed_share_no_written_slot(plan):
    """Every assignment of 3 slots (or none) to three sequences: of those let through, no two touch a slot that one writes."""
    for ins in itertools.product((-1, 0, 1, 2), repeat=3):
        for outs in itertools.product((-1, 0, 1, 2), repeat=3):
            ok = [not any(plan.slot_conflict(i, outs[i], j, ins[j], outs[j]) for j in range(3)) for i in range(3)]
            for i in range(3):
                if not ok[i] or outs[i] < 0:
                    continue
                for j in range(3):
                    if j != i:
                        assert ins[j] != outs[i] and not (ok[j] and outs[j] == outs[i])
            # what conflicts with nothing is let through
            for i in range(3):
                if outs[i] < 0 or all(outs[i] not in (ins[j], outs[j]) for j in range(3) if j != i):
                    assert ok[i]


def test_slots_outside_the_pool_are_found(plan):
    assert plan.slot_pair(4, -1, -1) == 0 and plan.slot_pair(4, 3, 0) == 0
    for a, b in ((-2, 0), (4, 0), (0, 4), (0, -2), (1 << 30, 0), (0, -(1 << 31))):
        assert plan.slot_pair(4, a, b) != 0
