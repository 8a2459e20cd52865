"""The C ABI of norms, 8-bit caches and shared beginnings: what it refuses before any device call (CPU)."""
import ctypes
import re

import pytest
import torch

import qe_mixer
import qe_moe


def test_null_arguments():
    lib = qe_mixer.load()
    b, c, c8, n, s = qe_mixer._Batch(), qe_mixer._Cache(), qe_mixer._Cache8(), qe_mixer._Norm(), qe_mixer._Shared()
    rows = (16, 64, 16, 64, 16, 64, None, 16, 64, None)
    assert lib.qe_attn_append_normed(None, b, c, n, 2, *rows) == qe_moe.QE_ERR_ARG
    assert lib.qe_attn_append8(None, b, c8, n, 2, *rows) == qe_moe.QE_ERR_ARG
    assert lib.qe_attn_append8(None, None, c8, None, 2, *rows) == qe_moe.QE_ERR_ARG
    assert lib.qe_attn_read8(None, b, c8, 16, 64, 16, 64, None) == qe_moe.QE_ERR_ARG
    assert lib.qe_attn_prompt8(None, None, c8, 16, 64, 16, 64, None) == qe_moe.QE_ERR_ARG
    assert lib.qe_attn_decode8(None, b, c8, 16, 64, 16, 64, None) == qe_moe.QE_ERR_ARG
    assert lib.qe_attn_decode_shared(None, b, s, c, 16, 64, 16, 64, None) == qe_moe.QE_ERR_ARG
    assert lib.qe_attn_decode8_shared(None, b, None, c8, 16, 64, 16, 64, None) == qe_moe.QE_ERR_ARG
    assert b"qe_attn_decode8_shared" in lib.qe_moe_last_error()


def test_constants_match_the_header():
    text = re.sub(r"/\*.*?\*/", "", open(qe_mixer.HEADER).read(), flags=re.S)
    assert int(re.search(r"#define QE_I8 (\d+)", text).group(1)) == qe_mixer.CODES[torch.int8]
    assert int(re.search(r"#define QE_F8 (\d+)", text).group(1)) == qe_mixer.CODES[torch.float8_e4m3fn]


def test_tensors_that_are_no_cache_norm_or_group():
    kc, s = torch.zeros(2, 1, 16, 64, dtype=torch.int8), torch.zeros(2, 1, 16)
    assert qe_mixer.Cache8(kc, kc.clone(), s, s.clone()).c.n_pages == 2
    for bad in (dict(kc=kc.short()), dict(vc=kc[:, :, :8]), dict(vc=kc.view(torch.float8_e4m3fn)), dict(k_scale=s.double()), dict(v_scale=s[..., None]),
                dict(kc=kc[0], vc=kc[0], k_scale=s[0], v_scale=s[0])):
        with pytest.raises(ValueError):
            qe_mixer.Cache8(**{**dict(kc=kc, vc=kc, k_scale=s, v_scale=s), **bad})
    for q, k in ((torch.ones(64, dtype=torch.bfloat16), None), (torch.ones(64), torch.ones(128)), (torch.ones(2, 64), None)):
        with pytest.raises(ValueError):
            qe_mixer.Norms(q, k)
    with pytest.raises(ValueError, match="32 bits"):
        qe_mixer.Shared(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), max_prefix=1 << 32)
    with pytest.raises(ValueError):
        qe_mixer.Shared(torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


def test_structs_have_the_headers_layout(tmp_path):
    """Sizes and offsets of the ctypes structures against a C compiler's."""
    import os
    import subprocess

    pairs = {"qe_kv_cache8": qe_mixer._Cache8, "qe_attn_norm": qe_mixer._Norm, "qe_attn_shared": qe_mixer._Shared}
    lines = [f'printf("%zu\\n", sizeof({n}));' + "".join(f'printf("%zu\\n", offsetof({n}, {f[0]}));' for f in t._fields_) for n, t in pairs.items()]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "qe_mixer.h"\nint main(void) {' + "".join(lines) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.dirname(qe_mixer.HEADER), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = [x for t in pairs.values() for x in (ctypes.sizeof(t), *(getattr(t, f[0]).offset for f in t._fields_))]
    assert got == want
