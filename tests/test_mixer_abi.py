"""The token mixers' C ABI: its symbols, and what it refuses before any device call (CPU)."""
import ctypes
import re

import pytest

import qe_mixer
import qe_moe

FINE = dict(q_heads=16, kv_heads=2, head_dim=256, page=256, type=2, scale=0.0, rotary=64, theta=1e7, sections=(11, 11, 10), interleaved=1)
DELTA = dict(k_heads=16, v_heads=32, dim_k=128, dim_v=128, type=0, l2norm=1, scale=0.0, t_max=64, seqs_max=4)


def _attn(**change):
    d = {**FINE, **change}
    d["sections"] = (ctypes.c_int * 3)(*d["sections"])
    h = ctypes.c_void_p()
    return qe_mixer.load().qe_attn_create(0, ctypes.byref(qe_mixer._AttnDesc(**d)), ctypes.byref(h))


def test_every_declared_symbol_is_exported_and_bound():
    lib = qe_mixer.load()
    text = re.sub(r"/\*.*?\*/", "", open(qe_mixer.HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(qe_(?:attn|delta)_\w+)\s*\(", text))
    assert names == set(qe_mixer._SIGNATURES)
    for n in names:
        assert hasattr(lib, n), n
    assert int(re.search(r"#define QE_ATTN_GROUP_MAX (\d+)", text).group(1)) == qe_mixer.QE_ATTN_GROUP_MAX
    for torch_type, value in qe_mixer.TYPES.items():
        name = {"torch.float32": "QE_F32", "torch.float16": "QE_F16", "torch.bfloat16": "QE_BF16"}[str(torch_type)]
        assert int(re.search(r"#define %s (\d+)" % name, text).group(1)) == value


@pytest.mark.parametrize("change", [
    dict(q_heads=15), dict(q_heads=34, kv_heads=2), dict(q_heads=0), dict(kv_heads=0), dict(kv_heads=257, q_heads=257), dict(head_dim=96),
    dict(head_dim=512), dict(page=8), dict(page=48), dict(page=512), dict(page=0), dict(type=0), dict(type=3), dict(scale=-1.0),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(rotary=-16), dict(rotary=24), dict(rotary=272), dict(theta=1.0),
    dict(theta=float("nan")), dict(theta=float("inf")), dict(sections=(11, 11, 11)), dict(sections=(32, -1, 1)),
    dict(sections=(0, 16, 16)), dict(sections=(9, 12, 11)), dict(sections=(0, 0, 0)),
])
def test_attention_geometries_that_are_refused(change):
    assert _attn(**change) == qe_moe.QE_ERR_ARG
    assert b"qe_attn_create" in qe_mixer.load().qe_moe_last_error()


@pytest.mark.parametrize("change", [
    dict(k_heads=0), dict(v_heads=24), dict(v_heads=0), dict(v_heads=2048, k_heads=2048), dict(dim_k=96), dict(dim_v=256), dict(type=5),
    dict(scale=-1.0), dict(scale=float("nan")), dict(t_max=0), dict(t_max=(1 << 20) + 1), dict(seqs_max=0), dict(seqs_max=65536),
])
def test_delta_geometries_that_are_refused(change):
    lib, h = qe_mixer.load(), ctypes.c_void_p()
    d = qe_mixer._DeltaDesc(**{**DELTA, **change})
    assert lib.qe_delta_create(0, ctypes.byref(d), ctypes.byref(h)) == qe_moe.QE_ERR_ARG
    assert b"qe_delta_create" in lib.qe_moe_last_error()


def test_sizes_beyond_32_bits_are_refused_by_the_binding():
    """ctypes would cut them: a page of 2^32 + 256 positions, say, to one of 256."""
    far = 1 << 32
    fine = dict(q_heads=16, kv_heads=2, head_dim=256, page=256, rotary=64, theta=1e7, sections=(11, 11, 10))
    for change in (dict(page=far + 256), dict(q_heads=far + 16), dict(rotary=far + 64), dict(sections=(far + 11, 11, 10)), dict(head_dim=256 - far)):
        with pytest.raises(ValueError, match="32 bits"):
            qe_mixer.Attention(**{**fine, **change})
    for change in (dict(t_max=far + 64), dict(seqs_max=far + 1), dict(v_heads=far + 32)):
        with pytest.raises(ValueError, match="32 bits"):
            qe_mixer.GatedDelta(**{**dict(k_heads=16, v_heads=32, dim_k=128, dim_v=128), **change})


def test_null_arguments():
    lib, h = qe_mixer.load(), ctypes.c_void_p()
    assert lib.qe_attn_create(0, None, ctypes.byref(h)) == qe_moe.QE_ERR_ARG
    assert lib.qe_delta_create(0, None, ctypes.byref(h)) == qe_moe.QE_ERR_ARG
    assert lib.qe_attn_destroy(None) == 0 and lib.qe_delta_destroy(None) == 0
    b, c, a = qe_mixer._Batch(), qe_mixer._Cache(), qe_mixer._DeltaArgs()
    assert lib.qe_attn_append(None, b, c, 2, 16, 64, 16, 64, 16, 64, None, 16, 64, None) == qe_moe.QE_ERR_ARG
    assert lib.qe_attn_prompt(None, None, c, 16, 64, 16, 64, None) == qe_moe.QE_ERR_ARG
    assert lib.qe_attn_decode(None, b, c, 16, 64, 16, 64, None) == qe_moe.QE_ERR_ARG
    assert lib.qe_attn_check(None, None) == qe_moe.QE_ERR_ARG
    assert lib.qe_delta_prompt(None, a, 16, None) == qe_moe.QE_ERR_ARG
    assert lib.qe_delta_decode(None, a, None) == qe_moe.QE_ERR_ARG
    assert lib.qe_delta_check(None, None) == qe_moe.QE_ERR_ARG
