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
and return without waiting.  A tensor of another type, shape or device raises ValueError; what
only the GPU can see leaves a code that ``status()`` returns.
"""
from __future__ import annotations

import ctypes as C
import math

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
        h = C.c_void_p()
        self._call(self.lib.rbt_paged_create(C.byref(h), C.byref(cfg), self.device.index or 0))
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
            return torch.cuda.current_stream(self.device).cuda_stream
        return stream if isinstance(stream, int) else stream.cuda_stream

    def _vector(self, t, n, name, dtype=torch.int32):
        """Address of a contiguous vector of n values on the pool's GPU (n None: of any length)."""
        if t.dtype is not dtype or t.device != self.device or t.dim() != 1 or (n is not None and t.shape[0] != n) or \
                not t.is_contiguous():
            raise ValueError(f"{name}: a contiguous {dtype} vector{'' if n is None else f' of {n}'} on {self.device} is "
                             f"wanted (got {t.dtype} {tuple(t.shape)} on {t.device})")
        return t.data_ptr()

    def _table(self, t, n):
        if t.dtype is not torch.int32 or t.device != self.device or t.dim() != 2 or t.shape[0] != n or \
                (t.shape[1] > 1 and t.stride(1) != 1):
            raise ValueError(f"table: int32 rows for {n} sequences on {self.device} are wanted "
                             f"(got {t.dtype} {tuple(t.shape)} on {t.device})")
        # only the row's own entries may be used: rows of another table lie between strided rows
        _want(t.stride(0) == t.shape[1] or n <= 1, "table: contiguous rows are wanted")
        return t.data_ptr(), t.shape[1]

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
        super().__init__(page, n_pages, ks[0].device, _cfg=RbtPagedConfig(len(ks), n_heads, kvh, hd, page, n_pages,
                                                                        _DTYPES[self.dtype]))
        for i, (a, b) in enumerate(zip(ks, vs)):
            self._call(self.lib.rbt_paged_bind_layer(self.handle, i, a.data_ptr(), b.data_ptr()))

    def _rows(self, t, heads, n, name, dtype):
        """Address and row stride of rows [n, heads, head dim] (heads of a row contiguous)."""
        shape = t.shape
        if t.dtype is not dtype or t.device != self.device or len(shape) != 3 or shape[0] != n or shape[1] != heads or \
                shape[2] != self.head_dim or t.stride(2) != 1 or (heads > 1 and t.stride(1) != self.head_dim):
            raise ValueError(f"{name}: {dtype} rows [{n}, {heads}, {self.head_dim}] on {self.device}, contiguous within "
                             f"a row, are wanted (got {t.dtype} {tuple(shape)}, strides {t.stride()}, on {t.device})")
        return t.data_ptr(), t.stride(0) if n > 1 else heads * self.head_dim

    def append(self, q, k, v, slot, pos, q_out, *, cos=None, sin=None, q_norm=None, k_norm=None, eps=1e-5, layer=0,
               stream=None):
        """k and v rows [n, kv heads, head dim] into their slots and q rows into q_out, after the
        whole-projection QK-norm (q_norm, k_norm) and RoPE (cos, sin [positions, head dim / 2])
        where given (rbt_paged_append_device)."""
        n = q.shape[0]
        _want(q.dtype in _DTYPES, f"q of {q.dtype}: float32 or bfloat16 are wanted")
        a = RbtPagedAppend()
        a.d_q, a.q_stride = self._rows(q, self.n_heads, n, "q", q.dtype)
        a.d_k, a.k_stride = self._rows(k, self.n_kv_heads, n, "k", q.dtype)
        a.d_v, a.v_stride = self._rows(v, self.n_kv_heads, n, "v", q.dtype)
        a.d_q_out, a.q_out_stride = self._rows(q_out, self.n_heads, n, "q_out", self.dtype)
        a.src_dtype, a.n_rows, a.eps = _DTYPES[q.dtype], n, eps
        a.d_slot = self._vector(slot, n, "slot", torch.int64)
        if pos is not None:
            a.d_pos = self._vector(pos, n, "pos")
        f32 = torch.float32
        if q_norm is not None:
            a.d_q_norm = self._vector(q_norm, self.n_heads * self.head_dim, "q_norm", f32)
        if k_norm is not None:
            a.d_k_norm = self._vector(k_norm, self.n_kv_heads * self.head_dim, "k_norm", f32)
        if cos is not None and sin is not None:
            for t, name in ((cos, "cos"), (sin, "sin")):
                _want(t.dtype is f32 and t.device == self.device and t.dim() == 2 and t.is_contiguous() and
                      t.shape == cos.shape and t.shape[1] * 2 == self.head_dim,
                      f"{name}: float32 [positions, {self.head_dim // 2}] on {self.device} is wanted")
            a.d_cos, a.d_sin, a.rope_len = cos.data_ptr(), sin.data_ptr(), cos.shape[0]
        else:
            _want(cos is None and sin is None, "cos and sin must both be given or both be None")
        self._call(self.lib.rbt_paged_append_device(self.handle, layer, C.byref(a), self._stream(stream)))

    def attention(self, q, out, cu, length, table, max_new, *, lse=None, causal=True, window=0, scale=None, layer=0,
                  stream=None):
        """out rows [n, heads, head dim] of the q rows' attention over their sequences' pages, and
        the rows' ln sum exp into lse [n, heads] where given (rbt_paged_attention_device).
        max_new: an upper bound of the sequences' new tokens; scale: 1/sqrt(head dim) if None."""
        n, n_seq = q.shape[0], length.shape[0]
        a = RbtPagedAttention()
        a.d_q, a.q_stride = self._rows(q, self.n_heads, n, "q", self.dtype)
        a.d_out, a.out_stride = self._rows(out, self.n_heads, n, "out", self.dtype)
        if lse is not None:
            _want(lse.dtype is torch.float32 and lse.device == self.device and tuple(lse.shape) == (n, self.n_heads) and
                  lse.is_contiguous(), f"lse: contiguous float32 [{n}, {self.n_heads}] on {self.device} is wanted")
            a.d_lse = lse.data_ptr()
        a.n_rows, a.n_seq, a.max_new = n, n_seq, max_new
        a.d_cu = self._vector(cu, n_seq + 1, "cu")
        a.d_len = self._vector(length, n_seq, "length")
        a.d_table, a.table_stride = self._table(table, n_seq)
        a.causal, a.window = bool(causal), window
        a.scale = 1.0 / math.sqrt(self.head_dim) if scale is None else scale
        self._call(self.lib.rbt_paged_attention_device(self.handle, layer, C.byref(a), self._stream(stream)))
