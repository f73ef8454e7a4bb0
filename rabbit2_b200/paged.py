"""Python binding of the paged KV cache of librbt_moe.so (rbt_paged_*, include/rbt_moe.h).

Plumbing over the C ABI for torch tensors, like moe.py and model.py.  ``PagedTables`` holds a
page pool's bookkeeping calls (``release``, ``plan``); ``PagedKv`` adds the caches of one or
more layers with ``append`` and ``attention``.  A serving step:

    kv = PagedKv(k_cache, v_cache, n_heads)   # [pages, kv heads, page size, head dim], per layer
    kv.release(length, done, table, free, n_free, held, n_mid)
    kv.plan(held, new, table, free, n_mid, length, n_free, cu, slot, pos)
    for each layer:
        kv.append(q, k, v, slot, pos, q, cos=cos, sin=sin, layer=l)
        kv.attention(q, out, cu, length, table, max_new, layer=l)

Lengths, tables, counts, offsets and positions are int32 tensors and slots int64, all on the
pool's GPU.  The calls run on the current stream of that GPU unless ``stream`` names another,
and return without waiting; they are for serving and record nothing for autograd.  A tensor of another type, shape or device raises ValueError; what
only the GPU can see leaves a code that ``status()`` returns.
"""
from __future__ import annotations

import ctypes as C
import math
import struct

import torch

from rabbit2_b200 import moe

MAX_SEQ = 2048


class RbtPagedConfig(C.Structure):
    _fields_ = [("n_layers", C.c_int32), ("n_heads", C.c_int32), ("n_kv_heads", C.c_int32), ("head_dim", C.c_int32),
                ("page_size", C.c_int32), ("n_pages", C.c_int32), ("dtype", C.c_int32)]


class RbtPagedAppend(C.Structure):
    _fields_ = [("d_q", C.c_void_p), ("d_k", C.c_void_p), ("d_v", C.c_void_p),
                ("q_stride", C.c_int64), ("k_stride", C.c_int64), ("v_stride", C.c_int64),
                ("src_dtype", C.c_int32), ("n_rows", C.c_int32), ("d_slot", C.c_void_p), ("d_pos", C.c_void_p),
                ("d_q_norm", C.c_void_p), ("d_k_norm", C.c_void_p), ("eps", C.c_float), ("rope_len", C.c_int32),
                ("d_cos", C.c_void_p), ("d_sin", C.c_void_p), ("d_q_out", C.c_void_p), ("q_out_stride", C.c_int64)]


class RbtPagedAttention(C.Structure):
    _fields_ = [("d_q", C.c_void_p), ("d_out", C.c_void_p), ("d_lse", C.c_void_p),
                ("q_stride", C.c_int64), ("out_stride", C.c_int64),
                ("n_rows", C.c_int32), ("n_seq", C.c_int32), ("max_new", C.c_int32),
                ("d_cu", C.c_void_p), ("d_len", C.c_void_p), ("d_table", C.c_void_p),
                ("table_stride", C.c_int32), ("causal", C.c_int32), ("window", C.c_int32), ("scale", C.c_float)]


_DTYPES = {torch.float32: moe.DT_F32, torch.bfloat16: moe.DT_BF16}
_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32
# the argument structs, packed in one call (a ctypes Structure costs a call per field)
_APPEND = struct.Struct("@QQQqqqiiQQQQfiQQQq")
_ATTENTION = struct.Struct("@QQQqqiiiQQQiiif")
assert _APPEND.size == C.sizeof(RbtPagedAppend) and _ATTENTION.size == C.sizeof(RbtPagedAttention)
_raw_stream = torch._C._cuda_getCurrentRawStream


def _want(ok, what):
    if not ok:
        raise ValueError(what)


class PagedTables:
    """Block tables of a pool of ``n_pages`` pages of ``page_size`` positions."""

    def __init__(self, page_size, n_pages, device=None, *, _cfg=None):
        self.lib = moe.load_library()
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.page_size, self.n_pages = page_size, n_pages
        cfg = _cfg or RbtPagedConfig(0, 0, 0, 0, page_size, n_pages, 0)
        if self.device.index is None:
            self.device = torch.device(self.device.type, torch.cuda.current_device())
        self.index = self.device.index
        h = C.c_void_p()
        self._call(self.lib.rbt_paged_create(C.byref(h), C.byref(cfg), self.index))
        self.handle = h.value

    def _call(self, ok):
        if not ok:
            raise moe.RbtMoeError(self.lib.rbt_moe_last_error().decode() or "call failed")

    def close(self):
        if getattr(self, "handle", None):
            self.lib.rbt_paged_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def status(self):
        """The status word of the calls so far (0: nothing went wrong), cleared; synchronises."""
        v = C.c_uint(0)
        self._call(self.lib.rbt_paged_status(self.handle, C.byref(v)))
        return v.value

    def _stream(self, stream):
        if stream is None:
            return _raw_stream(self.index)
        return stream if isinstance(stream, int) else stream.cuda_stream

    def _vector(self, t, n, name, dtype=_I32):
        """Address of a contiguous vector of n values on the pool's GPU (n None: of any length)."""
        if t.dtype is not dtype or t.get_device() != self.index or t.dim() != 1 or \
                (n is not None and t.numel() != n) or not t.is_contiguous():
            raise ValueError(f"{name}: a contiguous {dtype} vector{'' if n is None else f' of {n}'} on {self.device} is "
                             f"wanted (got {t.dtype} {tuple(t.shape)} on {t.device})")
        return t.data_ptr()

    def _table(self, t, n):
        shape = t.shape
        if t.dtype is not _I32 or t.get_device() != self.index or len(shape) != 2 or shape[0] != n or \
                not t.is_contiguous():
            raise ValueError(f"table: contiguous int32 rows for {n} sequences on {self.device} are wanted "
                             f"(got {t.dtype} {tuple(shape)} on {t.device})")
        return t.data_ptr(), shape[1]

    def release(self, length, done, table, free, n_free, length_out, n_free_out, stream=None):
        """Pages of the sequences with done != 0 back to the end of the free list
        (rbt_paged_release_device)."""
        n = length.shape[0]
        tp, ts = self._table(table, n)
        v = self._vector
        self._call(self.lib.rbt_paged_release_device(
            self.handle, n, v(length, n, "length"), v(done, n, "done"), tp, ts, v(free, None, "free"), free.shape[0],
            v(n_free, 1, "n_free"), v(length_out, n, "length_out"), v(n_free_out, 1, "n_free_out"),
            self._stream(stream)))

    def plan(self, length, new, table, free, n_free, length_out, n_free_out, cu, slot, pos, stream=None):
        """Pages from the end of the free list for ``new`` tokens of each sequence; their row
        offsets, slots and positions (rbt_paged_plan_device).  Rows of slot/pos past the new
        tokens get slot -1."""
        n = length.shape[0]
        tp, ts = self._table(table, n)
        v = self._vector
        rows = slot.shape[0]
        self._call(self.lib.rbt_paged_plan_device(
            self.handle, n, v(length, n, "length"), v(new, n, "new"), tp, ts, v(free, None, "free"),
            v(n_free, 1, "n_free"), rows, v(length_out, n, "length_out"), v(n_free_out, 1, "n_free_out"),
            v(cu, n + 1, "cu"), v(slot, rows, "slot", torch.int64), v(pos, rows, "pos"), self._stream(stream)))


class PagedKv(PagedTables):
    """The caches of one layer ([pages, kv heads, page size, head dim]) or of several (a list of
    those, or one more leading dimension) and the calls on them."""

    def __init__(self, k, v, n_heads):
        ks, vs = (list(t) if isinstance(t, (list, tuple)) or t.dim() == 5 else [t] for t in (k, v))
        _want(len(ks) > 0 and len(ks) == len(vs), "as many k caches as v caches are wanted")
        n_pages, kvh, page, hd = ks[0].shape
        for t in ks + vs:
            _want(t.shape == ks[0].shape and t.dtype == ks[0].dtype and t.device == ks[0].device and
                  t.is_contiguous() and t.is_cuda,
                  "the caches must be contiguous CUDA tensors of one shape, type and device")
        _want(ks[0].dtype in _DTYPES, f"caches of {ks[0].dtype}: float32 or bfloat16 are wanted")
        self.k, self.v, self.dtype = ks, vs, ks[0].dtype
        self.n_heads, self.n_kv_heads, self.head_dim = n_heads, kvh, hd
        self.scale = 1.0 / math.sqrt(hd)
        super().__init__(page, n_pages, ks[0].device, _cfg=RbtPagedConfig(len(ks), n_heads, kvh, hd, page, n_pages,
                                                                        _DTYPES[self.dtype]))
        for i, (a, b) in enumerate(zip(ks, vs)):
            self._call(self.lib.rbt_paged_bind_layer(self.handle, i, a.data_ptr(), b.data_ptr()))

    def _rows(self, t, heads, n, name, dtype):
        """Address and row stride of rows [n, heads, head dim] (heads of a row contiguous)."""
        hd = self.head_dim
        if t.dtype is not dtype or t.get_device() != self.index or t.shape != (n, heads, hd):
            raise ValueError(self._rows_wanted(t, heads, n, name, dtype))
        row, head, one = t.stride()
        if one != 1 or (head != hd and heads > 1):
            raise ValueError(self._rows_wanted(t, heads, n, name, dtype))
        return t.data_ptr(), row if n > 1 else heads * hd

    def _rows_wanted(self, t, heads, n, name, dtype):
        return (f"{name}: {dtype} rows [{n}, {heads}, {self.head_dim}] on {self.device}, contiguous within a row, are "
                f"wanted (got {t.dtype} {tuple(t.shape)}, strides {t.stride()}, on {t.device})")

    def append(self, q, k, v, slot, pos, q_out, *, cos=None, sin=None, q_norm=None, k_norm=None, eps=1e-5, layer=0,
               stream=None):
        """k and v rows [n, kv heads, head dim] into their slots and q rows into q_out, after the
        whole-projection QK-norm (q_norm, k_norm) and RoPE (cos, sin [positions, head dim / 2])
        where given (rbt_paged_append_device)."""
        n, dt, v32 = q.shape[0], q.dtype, self._vector
        src = _DTYPES.get(dt)
        _want(src is not None, f"q of {dt}: float32 or bfloat16 are wanted")
        qp, qs = self._rows(q, self.n_heads, n, "q", dt)
        kp, ks = self._rows(k, self.n_kv_heads, n, "k", dt)
        vp, vs = self._rows(v, self.n_kv_heads, n, "v", dt)
        op, os = self._rows(q_out, self.n_heads, n, "q_out", self.dtype)
        qn = 0 if q_norm is None else v32(q_norm, self.n_heads * self.head_dim, "q_norm", _F32)
        kn = 0 if k_norm is None else v32(k_norm, self.n_kv_heads * self.head_dim, "k_norm", _F32)
        cp = sp = angles = 0
        if cos is not None or sin is not None:
            _want(cos is not None and sin is not None, "cos and sin must both be given or both be None")
            for t, name in ((cos, "cos"), (sin, "sin")):
                _want(t.dtype is _F32 and t.get_device() == self.index and t.shape == cos.shape and t.dim() == 2 and
                      t.shape[1] * 2 == self.head_dim and t.is_contiguous(),
                      f"{name}: contiguous float32 [positions, {self.head_dim // 2}] on {self.device} is wanted")
            cp, sp, angles = cos.data_ptr(), sin.data_ptr(), cos.shape[0]
        a = _APPEND.pack(qp, kp, vp, qs, ks, vs, src, n, v32(slot, n, "slot", _I64),
                         0 if pos is None else v32(pos, n, "pos"), qn, kn, eps, angles, cp, sp, op, os)
        self._call(self.lib.rbt_paged_append_device(self.handle, layer, a, self._stream(stream)))

    def attention(self, q, out, cu, length, table, max_new, *, lse=None, causal=True, window=0, scale=None, layer=0,
                  stream=None):
        """out rows [n, heads, head dim] of the q rows' attention over their sequences' pages, and
        the rows' ln sum exp into lse [n, heads] where given (rbt_paged_attention_device).
        max_new: an upper bound of the sequences' new tokens; scale: 1/sqrt(head dim) if None."""
        n, n_seq = q.shape[0], length.shape[0]
        qp, qs = self._rows(q, self.n_heads, n, "q", self.dtype)
        op, os = self._rows(out, self.n_heads, n, "out", self.dtype)
        lp = 0
        if lse is not None:
            _want(lse.dtype is _F32 and lse.get_device() == self.index and lse.shape == (n, self.n_heads) and
                  lse.is_contiguous(), f"lse: contiguous float32 [{n}, {self.n_heads}] on {self.device} is wanted")
            lp = lse.data_ptr()
        tp, ts = self._table(table, n_seq)
        a = _ATTENTION.pack(qp, op, lp, qs, os, n, n_seq, max_new, self._vector(cu, n_seq + 1, "cu"),
                            self._vector(length, n_seq, "length"), tp, ts, 1 if causal else 0, window,
                            self.scale if scale is None else scale)
        self._call(self.lib.rbt_paged_attention_device(self.handle, layer, a, self._stream(stream)))
