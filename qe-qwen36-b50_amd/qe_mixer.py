"""ctypes binding of the token mixers (the C ABI in include/qe_mixer.h): attention over a
paged key-value cache, and the gated delta rule.

Tensors are torch tensors on the context's device; types, shapes and strides
are checked here, the rest by the library.  The calls run on the stream that is
given (None = the default stream) and return without a synchronisation: a tensor of
another stream is not freed before they have run (torch: record_stream).  There is
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
CODES = {torch.int8: 3, torch.float8_e4m3fn: 4}  # QE_I8, QE_F8

_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float


class _AttnDesc(ctypes.Structure):
    _fields_ = [("q_heads", _i32), ("kv_heads", _i32), ("head_dim", _i32), ("page", _i32), ("type", _i32), ("scale", _f32),
                ("rotary", _i32), ("theta", ctypes.c_double), ("sections", _i32 * 3), ("interleaved", _i32)]


class _Cache(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("n_pages", _i64)]


class _Batch(ctypes.Structure):
    _fields_ = [("n_seqs", _i32), ("n_tokens", _i32), ("cu_q", _vp), ("kv_len", _vp), ("table", _vp), ("table_stride", _i32),
                ("max_pages", _i32), ("max_len", _i32)]


class _Cache8(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("n_pages", _i64), ("type", _i32)]


class _Norm(ctypes.Structure):
    _fields_ = [("q_weight", _vp), ("k_weight", _vp), ("eps", _f32)]


class _Shared(ctypes.Structure):
    _fields_ = [("n_groups", _i32), ("seqs", _vp), ("prefix", _vp), ("max_prefix", _i32)]


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
    "qe_attn_append_normed": [_vp, ctypes.POINTER(_Batch), ctypes.POINTER(_Cache), ctypes.POINTER(_Norm), _i32, _vp, _i64, _vp, _i64, _vp,
                              _i64, _vp, _vp, _i64, _vp],
    "qe_attn_append8": [_vp, ctypes.POINTER(_Batch), ctypes.POINTER(_Cache8), ctypes.POINTER(_Norm), _i32, _vp, _i64, _vp, _i64, _vp, _i64,
                        _vp, _vp, _i64, _vp],
    "qe_attn_read8": [_vp, ctypes.POINTER(_Batch), ctypes.POINTER(_Cache8), _vp, _i64, _vp, _i64, _vp],
    "qe_attn_prompt": [_vp, ctypes.POINTER(_Batch), ctypes.POINTER(_Cache), _vp, _i64, _vp, _i64, _vp],
    "qe_attn_decode": [_vp, ctypes.POINTER(_Batch), ctypes.POINTER(_Cache), _vp, _i64, _vp, _i64, _vp],
    "qe_attn_prompt8": [_vp, ctypes.POINTER(_Batch), ctypes.POINTER(_Cache8), _vp, _i64, _vp, _i64, _vp],
    "qe_attn_decode8": [_vp, ctypes.POINTER(_Batch), ctypes.POINTER(_Cache8), _vp, _i64, _vp, _i64, _vp],
    "qe_attn_decode_shared": [_vp, ctypes.POINTER(_Batch), ctypes.POINTER(_Shared), ctypes.POINTER(_Cache), _vp, _i64, _vp, _i64, _vp],
    "qe_attn_decode8_shared": [_vp, ctypes.POINTER(_Batch), ctypes.POINTER(_Shared), ctypes.POINTER(_Cache8), _vp, _i64, _vp, _i64, _vp],
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


def _i32s(**sizes):
    """ctypes cuts integers to 32 bits without a word: a size beyond them would be another size."""
    for name, x in sizes.items():
        if not -(1 << 31) <= x < 1 << 31:
            _bad(f"{name} {x} does not fit 32 bits")


# The checks are written for their cost: a single token's call is a few microseconds of GPU work, and a
# tensor's shape, strides and device are fetched anew for every call.
def _on(x, device, name):
    if x.get_device() != device:
        _bad(f"{name} is on {x.device}, the context on cuda:{device}")


def _ints(x, shape, device, name):
    """Pointer of a contiguous int32 tensor of the given shape on the context's device."""
    if x.dtype is not torch.int32 or x.shape != shape or not x.is_contiguous() or x.get_device() != device:
        _on(x, device, name)
        _bad(f"{name}: a contiguous int32 tensor of shape {shape} is wanted, got {x.dtype} {tuple(x.shape)}")
    return x.data_ptr()


def _rows(x, heads, dim, dtype, device, name, tokens=None):
    """Pointer and token stride of [tokens, heads, dim], or [tokens, heads * dim], with contiguous tokens."""
    shape = x.shape
    if x.dtype is dtype and x.get_device() == device and (tokens is None or (shape and shape[0] == tokens)):
        if len(shape) == 3 and shape[1] == heads and shape[2] == dim:
            if x.is_contiguous():
                return x.data_ptr(), heads * dim
            stride = x.stride()
            if stride[2] == 1 and (stride[1] == dim or heads == 1):
                return x.data_ptr(), stride[0] if shape[0] > 1 else heads * dim
        elif len(shape) == 2 and shape[1] == heads * dim and x.stride(1) == 1:
            return x.data_ptr(), x.stride(0) if shape[0] > 1 else heads * dim
    _on(x, device, name)
    if x.dtype != dtype:
        _bad(f"{name} is {x.dtype}, {dtype} is wanted")
    _bad(f"{name}: [{'tokens' if tokens is None else tokens}, {heads}, {dim}] with contiguous tokens is wanted, "
         f"got {tuple(shape)} with strides {tuple(x.stride())}")


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
        _i32s(sequences=n, table_stride=stride, pages=table.shape[1], max_len=int(max_len))
        self.c = _Batch(n, n, None if cu_q is None else cu_q.data_ptr(), kv_len.data_ptr(), table.data_ptr(), stride,
                        table.shape[1], int(max_len))
        self._ref = ctypes.byref(self.c)

    def _with(self, n):
        """For tensors of n rows."""
        if self.n_tokens is not None:
            if self.n_tokens > n:
                _bad(f"the batch has {self.n_tokens} tokens, the tensors {n}")
            n = self.n_tokens
        self.c.n_tokens = n
        return self._ref


class Norms:
    """Norms of q's and k's heads before the rotation: float32 weights [head_dim] (None: not normed)."""

    def __init__(self, q_weight, k_weight, eps=1e-6):
        self.q_weight, self.k_weight = q_weight, k_weight
        self.device, self.dim = None, None
        for x, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
            if x is None:
                continue
            if x.dtype != torch.float32 or x.dim() != 1 or not x.is_contiguous() or (self.dim is not None and x.shape[0] != self.dim):
                _bad(f"{name}: contiguous float32 [head_dim] is wanted, got {x.dtype} {tuple(x.shape)}")
            if self.device is not None:
                _on(x, self.device, name)
            self.device, self.dim = x.get_device(), x.shape[0]
        self.c = _Norm(None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), eps)
        self._ref = ctypes.byref(self.c)


class Cache8:
    """An 8-bit cache: codes [pages, kv_heads, page, head_dim] of int8 or float8_e4m3fn, and float32 scales [pages, kv_heads,
    page] of their rows."""

    def __init__(self, kc, vc, k_scale, v_scale):
        if kc.dtype not in CODES:
            _bad(f"type {kc.dtype}: one of {', '.join(str(x) for x in CODES)} is taken")
        self.device, self.shape = kc.get_device(), tuple(kc.shape)
        for x, name, dtype, shape in ((kc, "k cache", kc.dtype, self.shape), (vc, "v cache", kc.dtype, self.shape),
                                      (k_scale, "k_scale", torch.float32, self.shape[:3]), (v_scale, "v_scale", torch.float32, self.shape[:3])):
            _on(x, self.device, name)
            if x.dtype != dtype or x.dim() != len(shape) or tuple(x.shape) != shape or len(self.shape) != 4 or not x.is_contiguous():
                _bad(f"{name}: contiguous {dtype} {shape} is wanted, got {x.dtype} {tuple(x.shape)}")
        self.kc, self.vc, self.k_scale, self.v_scale = kc, vc, k_scale, v_scale
        self.c = _Cache8(kc.data_ptr(), vc.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), kc.shape[0], CODES[kc.dtype])
        self._ref = ctypes.byref(self.c)


class Shared:
    """Groups of a batch's sequences that share their beginnings: int32 seqs [groups + 1], group g's first sequence and one
    behind its last, and prefix [groups], how many positions it shares (in the pages of its first sequence).  Both may be
    updated in place between calls.  max_prefix: the greatest as far as is known, for choosing splits (its difference from the batch's
    max_len is what sequences are expected to have to themselves)."""

    def __init__(self, seqs, prefix, max_prefix=0):
        n, device = prefix.shape[0], prefix.get_device()
        _ints(prefix, (n,), device, "prefix")
        _ints(seqs, (n + 1,), device, "seqs")
        _i32s(groups=n, max_prefix=int(max_prefix))
        self.device, self.seqs, self.prefix = device, seqs, prefix
        self.c = _Shared(n, seqs.data_ptr(), prefix.data_ptr(), int(max_prefix))
        self._ref = ctypes.byref(self.c)


class Attention:
    """One attention geometry on one GPU: rotary positions and cache write, prompts, single tokens."""

    def __init__(self, q_heads, kv_heads, head_dim, page, dtype=torch.bfloat16, rotary=0, theta=1e4, sections=None,
                 interleaved=False, scale=0.0, device=0):
        lib = load()
        s = tuple(sections) if sections is not None else (rotary // 2,)
        if len(s) > 3:
            _bad(f"sections {s}: at most three axes")
        s += (0,) * (3 - len(s))
        _i32s(q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, page=page, rotary=rotary, time=s[0], height=s[1], width=s[2])
        desc = _AttnDesc(q_heads, kv_heads, head_dim, page, _type(dtype, (torch.float16, torch.bfloat16)), scale, rotary, theta,
                         (_i32 * 3)(*s), int(interleaved))
        self.h = None
        h = _vp()
        _check(lib.qe_attn_create(device, ctypes.byref(desc), ctypes.byref(h)))
        self.h, self._lib = h, lib
        self.q_heads, self.kv_heads, self.head_dim, self.page, self.dtype, self.device = q_heads, kv_heads, head_dim, page, dtype, device
        self.n_axes = 3 if rotary and (s[1] or s[2]) else 1
        self._pages = (kv_heads, page, head_dim)
        self._c = _Cache()  # filled anew for every call
        self._ref = ctypes.byref(self._c)

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
        n = kc.shape
        if not (n == vc.shape and len(n) == 4 and n[1:] == self._pages and kc.dtype is self.dtype and vc.dtype is self.dtype
                and kc.is_contiguous() and vc.is_contiguous() and kc.get_device() == self.device and vc.get_device() == self.device):
            for x, name in ((kc, "k cache"), (vc, "v cache")):
                _on(x, self.device, name)
                if x.dtype != self.dtype or x.dim() != 4 or x.shape[1:] != self._pages or not x.is_contiguous():
                    _bad(f"{name}: contiguous {self.dtype} [pages, {', '.join(map(str, self._pages))}] is wanted, got {x.dtype} "
                         f"{tuple(x.shape)}")
            _bad(f"k and v caches of {kc.shape[0]} and {vc.shape[0]} pages")
        c = self._c
        c.k, c.v, c.n_pages = kc.data_ptr(), vc.data_ptr(), n[0]
        return self._ref

    def _batch(self, batch, n):
        if batch.device != self.device:
            _bad(f"the batch is on cuda:{batch.device}, the context on cuda:{self.device}")
        return batch._with(n)

    def _cache8(self, cache):
        if cache.shape[1:] != self._pages or cache.device != self.device:
            _on(cache.kc, self.device, "the cache")
            _bad(f"the cache: [pages, {', '.join(map(str, self._pages))}] is wanted, got {cache.shape}")
        return cache._ref

    def _norms(self, norms):
        if norms.dim is not None and (norms.dim != self.head_dim or norms.device != self.device):
            _bad(f"the norms are of {norms.dim} elements on cuda:{norms.device}, the heads of {self.head_dim} on cuda:{self.device}")
        return norms._ref

    def append(self, batch, q, k, v, kc, vc, q_out, pos=None, norms=None, stream=None):
        """Rotate q into q_out (both None: keys and values only), rotate k and write k and v to their pages.  norms: Norms of q and
        k before the rotation."""
        if norms is None:
            self._append(self._lib.qe_attn_append, (self._cache(kc, vc),), batch, q, k, v, q_out, pos, stream)
        else:
            self._append(self._lib.qe_attn_append_normed, (self._cache(kc, vc), self._norms(norms)), batch, q, k, v, q_out, pos, stream)

    def append8(self, batch, q, k, v, cache, q_out, pos=None, norms=None, stream=None):
        """The same to an 8-bit cache (Cache8)."""
        self._append(self._lib.qe_attn_append8, (self._cache8(cache), None if norms is None else self._norms(norms)), batch, q, k, v, q_out,
                     pos, stream)

    def _append(self, entry, where, batch, q, k, v, q_out, pos, stream):
        n, dt, dev = k.shape[0], k.dtype, self.device
        if dt is not self.dtype:
            _type(dt, (torch.float32, self.dtype))
        kp, ks = _rows(k, self.kv_heads, self.head_dim, dt, dev, "k")
        vp, vs = _rows(v, self.kv_heads, self.head_dim, dt, dev, "v", n)
        qp = op = None
        qs = os_ = 0
        if (q is None) != (q_out is None):
            _bad("q and q_out go together")
        if q is not None:
            qp, qs = _rows(q, self.q_heads, self.head_dim, dt, dev, "q", n)
            op, os_ = _rows(q_out, self.q_heads, self.head_dim, self.dtype, dev, "q_out", n)
        b = self._batch(batch, n)
        pp = None if pos is None else _ints(pos, (self.n_axes, batch.c.n_tokens), dev, "pos")
        rc = entry(self.h, b, *where, TYPES[dt], qp, qs, kp, ks, vp, vs, pp, op, os_, _stream(stream))
        if rc:
            _check(rc)

    def read8(self, batch, cache, k, v, stream=None):
        """The keys and values that an 8-bit cache holds for the positions of the batch's tokens (either may be None)."""
        x = k if k is not None else v
        if x is None:
            _bad("k and v are None")
        n = x.shape[0]
        kp = vp = None
        ks = vs = 0
        if k is not None:
            kp, ks = _rows(k, self.kv_heads, self.head_dim, self.dtype, self.device, "k", n)
        if v is not None:
            vp, vs = _rows(v, self.kv_heads, self.head_dim, self.dtype, self.device, "v", n)
        rc = self._lib.qe_attn_read8(self.h, self._batch(batch, n), self._cache8(cache), kp, ks, vp, vs, _stream(stream))
        if rc:
            _check(rc)

    def _attend(self, entry, batch, q, cache, out, stream, *shared):
        qp, qs = _rows(q, self.q_heads, self.head_dim, self.dtype, self.device, "q")
        n = q.shape[0]
        op, os_ = _rows(out, self.q_heads, self.head_dim, self.dtype, self.device, "out", n)
        rc = entry(self.h, self._batch(batch, n), *shared, cache, qp, qs, op, os_, _stream(stream))
        if rc:
            _check(rc)

    def prompt(self, batch, q, kc, vc, out, stream=None):
        """Causal attention of the batch's new tokens, which are in the cache, over their sequences."""
        self._attend(self._lib.qe_attn_prompt, batch, q, self._cache(kc, vc), out, stream)

    def decode(self, batch, q, kc, vc, out, stream=None):
        """The same for one new token per sequence (a batch without cu_q)."""
        self._attend(self._lib.qe_attn_decode, batch, q, self._cache(kc, vc), out, stream)

    def prompt8(self, batch, q, cache, out, stream=None):
        """prompt over an 8-bit cache (Cache8)."""
        self._attend(self._lib.qe_attn_prompt8, batch, q, self._cache8(cache), out, stream)

    def decode8(self, batch, q, cache, out, stream=None):
        """decode over an 8-bit cache (Cache8)."""
        self._attend(self._lib.qe_attn_decode8, batch, q, self._cache8(cache), out, stream)

    def _shared(self, shared):
        if shared.device != self.device:
            _bad(f"the groups are on cuda:{shared.device}, the context on cuda:{self.device}")
        return shared._ref

    def decode_shared(self, batch, shared, q, kc, vc, out, stream=None):
        """decode of sequences that share their beginnings (Shared)."""
        self._attend(self._lib.qe_attn_decode_shared, batch, q, self._cache(kc, vc), out, stream, self._shared(shared))

    def decode8_shared(self, batch, shared, q, cache, out, stream=None):
        """The same over an 8-bit cache (Cache8)."""
        self._attend(self._lib.qe_attn_decode8_shared, batch, q, self._cache8(cache), out, stream, self._shared(shared))

    def check(self, stream=None):
        """Synchronise `stream`; raise QeError if a kernel met a bad length or page."""
        _check(self._lib.qe_attn_check(self.h, _stream(stream)))


class GatedDelta:
    """One gated-delta-rule geometry on one GPU, with scratch for prompts of up to t_max tokens in seqs_max sequences."""

    def __init__(self, k_heads, v_heads, dim_k, dim_v, dtype=torch.float32, t_max=8192, seqs_max=64, l2norm=True, scale=0.0,
                 device=0):
        lib = load()
        _i32s(k_heads=k_heads, v_heads=v_heads, dim_k=dim_k, dim_v=dim_v, t_max=t_max, seqs_max=seqs_max)
        desc = _DeltaDesc(k_heads, v_heads, dim_k, dim_v, _type(dtype, tuple(TYPES)), int(l2norm), scale, t_max, seqs_max)
        self.h = None
        h = _vp()
        _check(lib.qe_delta_create(device, ctypes.byref(desc), ctypes.byref(h)))
        self.h, self._lib = h, lib
        self.k_heads, self.v_heads, self.dim_k, self.dim_v, self.dtype, self.device = k_heads, v_heads, dim_k, dim_v, dtype, device
        self._state = (v_heads, dim_k, dim_v)
        self._a = _DeltaArgs()  # filled anew for every call
        self._ref = ctypes.byref(self._a)

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
        n, dev, dt = q.shape[0], self.device, self.dtype
        a = self._a
        a.n_seqs, a.n_tokens = n_seqs, n
        a.q, a.q_stride = _rows(q, self.k_heads, self.dim_k, dt, dev, "q")
        a.k, a.k_stride = _rows(k, self.k_heads, self.dim_k, dt, dev, "k", n)
        a.v, a.v_stride = _rows(v, self.v_heads, self.dim_v, dt, dev, "v", n)
        a.out, a.out_stride = _rows(out, self.v_heads, self.dim_v, dt, dev, "out", n)
        for x, name in ((g, "g"), (beta, "beta")):
            if x.dtype is not torch.float32 or x.shape != (n, self.v_heads) or not x.is_contiguous() or x.get_device() != dev:
                _on(x, dev, name)
                _bad(f"{name}: contiguous float32 [{n}, {self.v_heads}] is wanted, got {x.dtype} {tuple(x.shape)}")
        p = pool.shape
        if pool.dtype is not torch.float32 or len(p) != 4 or p[1:] != self._state or not pool.is_contiguous() or pool.get_device() != dev:
            _on(pool, dev, "pool")
            _bad(f"pool: contiguous float32 [slots, {', '.join(map(str, self._state))}] is wanted, got {pool.dtype} {tuple(p)}")
        a.g, a.beta, a.pool, a.n_slots = g.data_ptr(), beta.data_ptr(), pool.data_ptr(), p[0]
        a.slots_in, a.slots_out = _ints(slots_in, (n_seqs,), dev, "slots_in"), _ints(slots_out, (n_seqs,), dev, "slots_out")
        return self._ref

    def prompt(self, q, k, v, g, beta, pool, slots_in, slots_out, cu, out, stream=None):
        """Packed prompts: sequence i is rows cu[i] .. cu[i + 1] - 1; its state comes from pool[slots_in[i]] (-1: zeros) and
        goes to pool[slots_out[i]] (-1: nowhere)."""
        n = slots_in.shape[0]
        a = self._args(n, q, k, v, g, beta, pool, slots_in, slots_out, out)
        rc = self._lib.qe_delta_prompt(self.h, a, _ints(cu, (n + 1,), self.device, "cu"), _stream(stream))
        if rc:
            _check(rc)

    def decode(self, q, k, v, g, beta, pool, slots_in, slots_out, out, stream=None):
        """One token per sequence: row i is sequence i's."""
        rc = self._lib.qe_delta_decode(self.h, self._args(q.shape[0], q, k, v, g, beta, pool, slots_in, slots_out, out), _stream(stream))
        if rc:
            _check(rc)

    def check(self, stream=None):
        """Synchronise `stream`; raise QeError if a kernel met a bad slot or token offset."""
        _check(self._lib.qe_delta_check(self.h, _stream(stream)))
