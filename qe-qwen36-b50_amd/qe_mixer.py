"""ctypes binding of the token mixers (the C ABI in include/qe_mixer.h): attention over a
paged key-value cache, and the gated delta rule.

Tensors are torch tensors on the context's device; types, shapes and strides
are checked here, the rest by the library.  The calls run on the stream that is
given (None = the default stream) and return without a synchronisation.  There is
no fallback: without the library, LibraryMissing is raised.
"""
from __future__ import annotations

import ctypes
import os

import torch

import qe_moe
from qe_moe import QeError, _check, _stream  # noqa: F401  (QeError is what calls raise)

HEADER = os.path.join(os.path.dirname(qe_moe.HERE), "include", "qe_mixer.h")
QE_ATTN_GROUP_MAX = 16  # include/qe_mixer.h
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # QE_F32, QE_F16, QE_BF16

_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float


class _AttnDesc(ctypes.Structure):
    _fields_ = [("q_heads", _i32), ("kv_heads", _i32), ("head_dim", _i32), ("page", _i32), ("type", _i32), ("scale", _f32),
                ("rotary", _i32), ("theta", ctypes.c_double), ("sections", _i32 * 3), ("interleaved", _i32)]


class _Cache(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("n_pages", _i64)]


class _Batch(ctypes.Structure):
    _fields_ = [("n_seqs", _i32), ("n_tokens", _i32), ("cu_q", _vp), ("kv_len", _vp), ("table", _vp), ("table_stride", _i32),
                ("max_pages", _i32), ("max_len", _i32)]


class _DeltaDesc(ctypes.Structure):
    _fields_ = [("k_heads", _i32), ("v_heads", _i32), ("dim_k", _i32), ("dim_v", _i32), ("type", _i32), ("l2norm", _i32),
                ("scale", _f32), ("t_max", _i32), ("seqs_max", _i32)]


class _DeltaArgs(ctypes.Structure):
    _fields_ = [("n_seqs", _i32), ("n_tokens", _i32), ("q", _vp), ("k", _vp), ("v", _vp), ("q_stride", _i64), ("k_stride", _i64),
                ("v_stride", _i64), ("g", _vp), ("beta", _vp), ("pool", _vp), ("n_slots", _i64), ("slots_in", _vp),
                ("slots_out", _vp), ("out", _vp), ("out_stride", _i64)]


_SIGNATURES = {
    "qe_attn_create": [_i32, ctypes.POINTER(_AttnDesc), ctypes.POINTER(_vp)],
    "qe_attn_destroy": [_vp],
    "qe_attn_append": [_vp, ctypes.POINTER(_Batch), ctypes.POINTER(_Cache), _i32, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _i64,
                       _vp],
    "qe_attn_prompt": [_vp, ctypes.POINTER(_Batch), ctypes.POINTER(_Cache), _vp, _i64, _vp, _i64, _vp],
    "qe_attn_decode": [_vp, ctypes.POINTER(_Batch), ctypes.POINTER(_Cache), _vp, _i64, _vp, _i64, _vp],
    "qe_attn_check": [_vp, _vp],
    "qe_delta_create": [_i32, ctypes.POINTER(_DeltaDesc), ctypes.POINTER(_vp)],
    "qe_delta_destroy": [_vp],
    "qe_delta_prompt": [_vp, ctypes.POINTER(_DeltaArgs), _vp, _vp],
    "qe_delta_decode": [_vp, ctypes.POINTER(_DeltaArgs), _vp],
    "qe_delta_check": [_vp, _vp],
}


_bound = None


def load():
    global _bound
    lib = qe_moe.load()
    if _bound is not lib:
        for name, args in _SIGNATURES.items():
            f = getattr(lib, name)
            f.restype, f.argtypes = _i32, args
        _bound = lib
    return lib


def _bad(text):
    raise ValueError(text)


def _type(dtype, allowed):
    if dtype not in allowed:
        _bad(f"type {dtype}: one of {', '.join(str(x) for x in allowed)} is taken")
    return TYPES[dtype]


def _on(x, device, name):
    if x.device.type != "cuda" or x.device.index != device:
        _bad(f"{name} is on {x.device}, the context on cuda:{device}")


def _ints(x, shape, device, name):
    """A contiguous int32 tensor of the given shape (None = any) on the context's device."""
    _on(x, device, name)
    if x.dtype != torch.int32 or x.dim() != len(shape) or any(b is not None and a != b for a, b in zip(x.shape, shape)) \
            or not x.is_contiguous():
        _bad(f"{name}: a contiguous int32 tensor of shape {shape} is wanted, got {x.dtype} {tuple(x.shape)}")
    return x.data_ptr()


def _rows(x, heads, dim, dtype, device, name, tokens=None):
    """Pointer and token stride of [tokens, heads, dim], or [tokens, heads * dim], with contiguous tokens."""
    _on(x, device, name)
    if x.dtype != dtype:
        _bad(f"{name} is {x.dtype}, {dtype} is wanted")
    shape, stride = x.shape, x.stride()
    if tokens is not None and (len(shape) == 0 or shape[0] != tokens):
        _bad(f"{name} has shape {tuple(shape)}, {tokens} tokens are wanted")
    if len(shape) == 3 and shape[1] == heads and shape[2] == dim:
        fine = (stride[2] == 1 or dim == 1) and (stride[1] == dim or heads == 1)
    else:
        fine = len(shape) == 2 and shape[1] == heads * dim and stride[1] == 1
    if not fine:
        _bad(f"{name}: [{'tokens' if tokens is None else tokens}, {heads}, {dim}] with contiguous tokens is wanted, "
             f"got {tuple(shape)} with strides {tuple(stride)}")
    return x.data_ptr(), stride[0] if shape[0] > 1 else heads * dim


class Batch:
    """The sequences of an attention call: lengths and page tables in device memory, which the caller may update in
    place between calls (as a captured graph needs).  cu_q None: one new token per sequence."""

    def __init__(self, kv_len, table, cu_q=None, n_tokens=None, max_len=0):
        """kv_len int32 [n]; table int32 [n, pages]; cu_q int32 [n + 1].  n_tokens: rows that q, k, v and out have, taken
        from them if not given.  max_len: the longest kv_len as far as is known, for choosing splits."""
        n, device = kv_len.shape[0], kv_len.device.index
        _ints(kv_len, (n,), device, "kv_len")
        _on(table, device, "table")
        if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != n or (table.shape[1] > 1 and table.stride(1) != 1):
            _bad(f"table: int32 [{n}, pages] with contiguous rows is wanted, got {table.dtype} {tuple(table.shape)}")
        if cu_q is not None:
            _ints(cu_q, (n + 1,), device, "cu_q")
        self.device, self.kv_len, self.table, self.cu_q, self.n_tokens = device, kv_len, table, cu_q, n_tokens
        stride = table.stride(0) if n > 1 else table.shape[1]
        self.c = _Batch(n, n, None if cu_q is None else cu_q.data_ptr(), kv_len.data_ptr(), table.data_ptr(), stride,
                        table.shape[1], int(max_len))

    def _with(self, rows):
        n = rows.shape[0] if self.n_tokens is None else self.n_tokens
        if n > rows.shape[0]:
            _bad(f"the batch has {n} tokens, the tensors {rows.shape[0]}")
        self.c.n_tokens = n
        return ctypes.byref(self.c)


class Attention:
    """One attention geometry on one GPU: rotary positions and cache write, prompts, single tokens."""

    def __init__(self, q_heads, kv_heads, head_dim, page, dtype=torch.bfloat16, rotary=0, theta=1e4, sections=None,
                 interleaved=False, scale=0.0, device=0):
        lib = load()
        s = tuple(sections) if sections is not None else (rotary // 2,)
        if len(s) > 3:
            _bad(f"sections {s}: at most three axes")
        s += (0,) * (3 - len(s))
        desc = _AttnDesc(q_heads, kv_heads, head_dim, page, _type(dtype, (torch.float16, torch.bfloat16)), scale, rotary, theta,
                         (_i32 * 3)(*s), int(interleaved))
        self.h = None
        h = _vp()
        _check(lib.qe_attn_create(device, ctypes.byref(desc), ctypes.byref(h)))
        self.h, self._lib = h, lib
        self.q_heads, self.kv_heads, self.head_dim, self.page, self.dtype, self.device = q_heads, kv_heads, head_dim, page, dtype, device
        self.n_axes = 3 if rotary and (s[1] or s[2]) else 1

    def close(self):
        if self.h:
            self._lib.qe_attn_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _cache(self, kc, vc):
        want = (self.kv_heads, self.page, self.head_dim)
        for x, name in ((kc, "k cache"), (vc, "v cache")):
            _on(x, self.device, name)
            if x.dtype != self.dtype or x.dim() != 4 or x.shape[1:] != want or not x.is_contiguous():
                _bad(f"{name}: contiguous {self.dtype} [pages, {want[0]}, {want[1]}, {want[2]}] is wanted, got {x.dtype} {tuple(x.shape)}")
        if kc.shape[0] != vc.shape[0]:
            _bad(f"k and v caches of {kc.shape[0]} and {vc.shape[0]} pages")
        return ctypes.byref(_Cache(kc.data_ptr(), vc.data_ptr(), kc.shape[0]))

    def _batch(self, batch, rows):
        if batch.device != self.device:
            _bad(f"the batch is on cuda:{batch.device}, the context on cuda:{self.device}")
        return batch._with(rows)

    def append(self, batch, q, k, v, kc, vc, q_out, pos=None, stream=None):
        """Rotate q into q_out (both None: keys and values only), rotate k and write k and v to their pages."""
        n = k.shape[0]
        dt = k.dtype
        _type(dt, (torch.float32, self.dtype))
        kp, ks = _rows(k, self.kv_heads, self.head_dim, dt, self.device, "k")
        vp, vs = _rows(v, self.kv_heads, self.head_dim, dt, self.device, "v", n)
        qp = qs = op = os_ = None
        if (q is None) != (q_out is None):
            _bad("q and q_out go together")
        if q is not None:
            qp, qs = _rows(q, self.q_heads, self.head_dim, dt, self.device, "q", n)
            op, os_ = _rows(q_out, self.q_heads, self.head_dim, self.dtype, self.device, "q_out", n)
        b = self._batch(batch, k)
        pp = None if pos is None else _ints(pos, (self.n_axes, batch.c.n_tokens), self.device, "pos")
        _check(self._lib.qe_attn_append(self.h, b, self._cache(kc, vc), TYPES[dt], qp, qs or 0, kp, ks, vp, vs, pp, op, os_ or 0,
                                        _stream(stream)))

    def _attend(self, entry, batch, q, kc, vc, out, stream):
        qp, qs = _rows(q, self.q_heads, self.head_dim, self.dtype, self.device, "q")
        op, os_ = _rows(out, self.q_heads, self.head_dim, self.dtype, self.device, "out", q.shape[0])
        _check(entry(self.h, self._batch(batch, q), self._cache(kc, vc), qp, qs, op, os_, _stream(stream)))

    def prompt(self, batch, q, kc, vc, out, stream=None):
        """Causal attention of the batch's new tokens, which are in the cache, over their sequences."""
        self._attend(self._lib.qe_attn_prompt, batch, q, kc, vc, out, stream)

    def decode(self, batch, q, kc, vc, out, stream=None):
        """The same for one new token per sequence (a batch without cu_q)."""
        self._attend(self._lib.qe_attn_decode, batch, q, kc, vc, out, stream)

    def check(self, stream=None):
        """Synchronise `stream`; raise QeError if a kernel met a bad length or page."""
        _check(self._lib.qe_attn_check(self.h, _stream(stream)))


class GatedDelta:
    """One gated-delta-rule geometry on one GPU, with scratch for prompts of up to t_max tokens in seqs_max sequences."""

    def __init__(self, k_heads, v_heads, dim_k, dim_v, dtype=torch.float32, t_max=8192, seqs_max=64, l2norm=True, scale=0.0,
                 device=0):
        lib = load()
        desc = _DeltaDesc(k_heads, v_heads, dim_k, dim_v, _type(dtype, tuple(TYPES)), int(l2norm), scale, t_max, seqs_max)
        self.h = None
        h = _vp()
        _check(lib.qe_delta_create(device, ctypes.byref(desc), ctypes.byref(h)))
        self.h, self._lib = h, lib
        self.k_heads, self.v_heads, self.dim_k, self.dim_v, self.dtype, self.device = k_heads, v_heads, dim_k, dim_v, dtype, device

    def close(self):
        if self.h:
            self._lib.qe_delta_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _args(self, n_seqs, q, k, v, g, beta, pool, slots_in, slots_out, out):
        n, dev = q.shape[0], self.device
        qp, qs = _rows(q, self.k_heads, self.dim_k, self.dtype, dev, "q")
        kp, ks = _rows(k, self.k_heads, self.dim_k, self.dtype, dev, "k", n)
        vp, vs = _rows(v, self.v_heads, self.dim_v, self.dtype, dev, "v", n)
        op, os_ = _rows(out, self.v_heads, self.dim_v, self.dtype, dev, "out", n)
        for x, name in ((g, "g"), (beta, "beta")):
            _on(x, dev, name)
            if x.dtype != torch.float32 or tuple(x.shape) != (n, self.v_heads) or not x.is_contiguous():
                _bad(f"{name}: contiguous float32 [{n}, {self.v_heads}] is wanted, got {x.dtype} {tuple(x.shape)}")
        _on(pool, dev, "pool")
        if pool.dtype != torch.float32 or pool.dim() != 4 or tuple(pool.shape[1:]) != (self.v_heads, self.dim_k, self.dim_v) \
                or not pool.is_contiguous():
            _bad(f"pool: contiguous float32 [slots, {self.v_heads}, {self.dim_k}, {self.dim_v}] is wanted, got {pool.dtype} "
                 f"{tuple(pool.shape)}")
        return _DeltaArgs(n_seqs, n, qp, kp, vp, qs, ks, vs, g.data_ptr(), beta.data_ptr(), pool.data_ptr(), pool.shape[0],
                          _ints(slots_in, (n_seqs,), dev, "slots_in"), _ints(slots_out, (n_seqs,), dev, "slots_out"), op, os_)

    def prompt(self, q, k, v, g, beta, pool, slots_in, slots_out, cu, out, stream=None):
        """Packed prompts: sequence i is rows cu[i] .. cu[i + 1] - 1; its state comes from pool[slots_in[i]] (-1: zeros) and
        goes to pool[slots_out[i]] (-1: nowhere)."""
        n = slots_in.shape[0]
        a = self._args(n, q, k, v, g, beta, pool, slots_in, slots_out, out)
        _check(self._lib.qe_delta_prompt(self.h, ctypes.byref(a), _ints(cu, (n + 1,), self.device, "cu"), _stream(stream)))

    def decode(self, q, k, v, g, beta, pool, slots_in, slots_out, out, stream=None):
        """One token per sequence: row i is sequence i's."""
        a = self._args(q.shape[0], q, k, v, g, beta, pool, slots_in, slots_out, out)
        _check(self._lib.qe_delta_decode(self.h, ctypes.byref(a), _stream(stream)))

    def check(self, stream=None):
        """Synchronise `stream`; raise QeError if a kernel met a bad slot or token offset."""
        _check(self._lib.qe_delta_check(self.h, _stream(stream)))
