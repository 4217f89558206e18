"""ctypes binding of the token-step operators of libhipvoc.so (include/hipvoc_ops.h).

``HipOps.open(device)`` gives a handle; its methods take torch tensors of that device and enqueue on torch's current stream
of it, so they can be captured into a graph with the rest of a step.  They allocate their results (and a workspace, where one
is needed) as torch operations do; the C entry points take the caller's memory.  A refused call raises HipVocError before
anything is launched; what only the device can see (a page number, a length) is raised by ``sync()``.

There is NO fallback: if the shared library is missing or no HIP device is present, opening raises.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

from .hipvoc import HipVocError, load_library

OPS_EXPORTS = [
    "hipvoc_ops_open", "hipvoc_ops_sync", "hipvoc_kv_write", "hipvoc_kv_read", "hipvoc_attention_workspace",
    "hipvoc_attention", "hipvoc_add_rmsnorm", "hipvoc_q4_matvec",
]

T_F32, T_F16, T_BF16, T_INT8, T_E4M3 = 0, 1, 2, 3, 4      # include/hipvoc_ops.h: HIPVOC_T_*


class _Cache(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("page_stride", C.c_int64),
                ("n_pages", C.c_int32), ("kv_heads", C.c_int32), ("page", C.c_int32), ("head_dim", C.c_int32), ("dtype", C.c_int32)]


class _Rows(C.Structure):
    _fields_ = [("table", C.c_void_p), ("cu", C.c_void_p), ("first", C.c_void_p), ("table_stride", C.c_int64),
                ("table_width", C.c_int32), ("n_seqs", C.c_int32)]


_bound = False


def _lib():
    global _bound
    L = load_library()
    if not _bound:
        vp, i64, i32, f32 = C.c_void_p, C.c_int64, C.c_int, C.c_float
        L.hipvoc_ops_open.restype = vp
        L.hipvoc_ops_open.argtypes = [i32]
        L.hipvoc_ops_sync.argtypes = [vp, vp]
        L.hipvoc_kv_write.argtypes = [vp, vp, vp, vp, i64, i64, i32, vp, i32, vp]
        L.hipvoc_kv_read.argtypes = [vp, vp, vp, vp, i64, i64, i32, vp, i32, vp]
        L.hipvoc_attention_workspace.restype = C.c_size_t
        L.hipvoc_attention_workspace.argtypes = [vp, i32, i32, i32, i32]
        L.hipvoc_attention.argtypes = [vp, vp, vp, i64, vp, i64, vp, i32, i32, vp, i64, i32, vp, i32, i32, i32, f32, vp, C.c_size_t, vp]
        L.hipvoc_add_rmsnorm.argtypes = [vp, vp, i64, vp, i64, vp, vp, i64, vp, i64, vp, i32, i32, i32, f32, i32, i32, vp]
        L.hipvoc_q4_matvec.argtypes = [vp, vp, vp, vp, i32, i32, i32, vp, i64, i32, vp, i32, vp, i64, i32, i32, vp]
        _bound = True
    return L


torch = None
_types = {}                     # torch dtype -> HIPVOC_T_*


def _bind_torch():
    """The rest of the package needs no torch: it is imported when the first cache or handle is made."""
    global torch
    if torch is None:
        import torch as module
        _types.update({module.float32: T_F32, module.float16: T_F16, module.bfloat16: T_BF16, module.int8: T_INT8, module.float8_e4m3fn: T_E4M3})
        torch = module


def _refuse(msg: str):
    raise HipVocError(-1, msg)


def _type(t) -> int:
    code = _types.get(t.dtype, -1)
    if code < 0:
        _refuse(f"unsupported dtype {t.dtype}")
    return code


class KvCache:
    """Names the tensors of a paged cache (hipvoc_kv_cache): k, v [n_pages, kv_heads, page, head_dim], contiguous within a page;
    k_scale, v_scale [n_pages, kv_heads, page] float32 for int8 / float8_e4m3fn caches."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        _bind_torch()
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            _refuse("k and v must be [n_pages, kv_heads, page, head_dim], alike in shape, type and device")
        n, heads, page, hd = k.shape
        inner = (page * hd, hd, 1)
        stride = k.stride(0) if n > 1 else heads * page * hd
        if k.stride()[1:] != inner or v.stride()[1:] != inner or (n > 1 and v.stride(0) != stride):
            _refuse("a page of k and of v must be contiguous, and their page strides equal")
        self.dtype = _type(k)
        if (self.dtype >= T_INT8) != (k_scale is not None) or (k_scale is None) != (v_scale is None):
            _refuse("an 8-bit cache needs k_scale and v_scale, any other has none")
        for s in (k_scale, v_scale):
            if s is not None and (tuple(s.shape) != (n, heads, page) or not s.is_contiguous() or _type(s) != T_F32 or s.device != k.device):
                _refuse("scales must be contiguous float32 [n_pages, kv_heads, page] on the cache's device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale          # kept alive
        self.device, self.kv_heads, self.page, self.head_dim, self.n_pages = k.device, heads, page, hd, n
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self._c = _Cache(ptr(k), ptr(v), ptr(k_scale), ptr(v_scale), stride, n, heads, page, hd, self.dtype)
        self._p = C.addressof(self._c)


class HipOps:
    """The operators of one token step on one MI355X."""

    def __init__(self, handle, lib, device: int):
        _bind_torch()
        self._h = handle
        self._L = lib
        self.device = torch.device("cuda", device)
        self._index = device

    @classmethod
    def open(cls, device: int = 0) -> "HipOps":
        L = _lib()
        h = L.hipvoc_ops_open(device)
        if not h:
            raise HipVocError(-6, L.hipvoc_last_error(None).decode())
        return cls(h, L, device)

    def close(self):
        if self._h:
            self._L.hipvoc_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _failed(self, rc: int):
        raise HipVocError(rc, self._L.hipvoc_last_error(self._h).decode() if self._h else "the handle is closed")

    @property
    def stream(self) -> int:
        """torch's current stream of the handle's device, where the calls are enqueued."""
        return torch._C._cuda_getCurrentRawStream(self._index)

    def sync(self):
        """Waits for the current stream and raises what the device found wrong since the last time."""
        rc = self._L.hipvoc_ops_sync(self._h, self.stream)
        if rc:
            self._failed(rc)

    # ---- what a call looks at in its tensors (a step makes these calls per layer: each attribute is asked for once) -----
    def _elsewhere(self, name, t):
        _refuse(f"{name} is on {t.device}, the handle on {self.device}")

    def _here(self, name, t):
        if t is not None and t.device != self.device:
            self._elsewhere(name, t)

    def _ints(self, name, t, n):
        """Address of a contiguous int32 vector of n values."""
        if t.dtype != torch.int32 or t.shape != (n,) or (n > 1 and t.stride(0) != 1):
            _refuse(f"{name} must be a contiguous int32 vector of {n}")
        if t.device != self.device:
            self._elsewhere(name, t)
        return t.data_ptr()

    def _table(self, t):
        """(address, stride, width, rows) of a page table."""
        shape = t.shape
        if t.dtype != torch.int32 or len(shape) != 2:
            _refuse("table must be int32 [seqs, pages]")
        stride = t.stride()
        if shape[1] > 1 and stride[1] != 1:
            _refuse("table must have contiguous rows")
        if t.device != self.device:
            self._elsewhere("table", t)
        return t.data_ptr(), stride[0], shape[1], shape[0]

    def _heads(self, name, t, heads, hd):
        """(rows, row stride) of [rows, heads, head_dim] with contiguous rows."""
        shape, stride = t.shape, t.stride()
        if len(shape) != 3 or shape[1] != heads or shape[2] != hd or stride[2] != 1 or (heads > 1 and stride[1] != hd):
            _refuse(f"{name} must be [rows, {heads}, {hd}] with contiguous rows")
        if t.device != self.device:
            self._elsewhere(name, t)
        rows = shape[0]
        if rows >> 31:
            _refuse(f"{name} has {rows} rows")
        return rows, stride[0] if rows > 1 else heads * hd

    def _matrix(self, name, t):
        """(rows, columns, row stride) of a matrix with contiguous rows."""
        shape = t.shape
        if len(shape) != 2:
            _refuse(f"{name} must be a matrix")
        rows, cols = shape
        stride = t.stride()
        if stride[1] != 1 and cols > 1:
            _refuse(f"{name} must have contiguous rows")
        if t.device != self.device:
            self._elsewhere(name, t)
        if rows >> 31 or cols >> 31:
            _refuse(f"{name} is {rows} by {cols}")
        return rows, cols, stride[0] if rows > 1 else cols

    # ---- the paged cache -----------------------------------------------------------------
    def kv_cache(self, k, v, k_scale=None, v_scale=None) -> KvCache:
        self._here("k", k)
        return KvCache(k, v, k_scale, v_scale)

    def _rows(self, table, cu, first):
        tp, stride, width, n = self._table(table)
        return _Rows(tp, self._ints("cu", cu, n + 1), self._ints("first", first, n), stride, width, n)

    def kv_write(self, cache: KvCache, k, v, table, cu, first):
        """k, v [rows, kv_heads, head_dim]: rows cu[b] .. cu[b+1] go to positions first[b] ... of sequence b (pages table[b])."""
        if cache.device != self.device:
            self._elsewhere("the cache", cache)
        n, ks = self._heads("k", k, cache.kv_heads, cache.head_dim)
        nv, vs = self._heads("v", v, cache.kv_heads, cache.head_dim)
        if n != nv or k.dtype != v.dtype:
            _refuse("k and v must be alike")
        r = self._rows(table, cu, first)
        rc = self._L.hipvoc_kv_write(self._h, cache._p, k.data_ptr(), v.data_ptr(), ks, vs, _type(k), C.addressof(r), n, self.stream)
        if rc:
            self._failed(rc)

    def kv_read(self, cache: KvCache, table, cu, first, n_rows: int, dtype=None, out: Optional[Tuple] = None):
        """The inverse: (k, v) [n_rows, kv_heads, head_dim] in `dtype` (default: the cache's own), or into the two tensors of `out`;
        rows at or behind cu[-1] are left as they were."""
        if cache.device != self.device:
            self._elsewhere("the cache", cache)
        if not 0 <= n_rows < 1 << 31:
            _refuse(f"n_rows {n_rows} is negative or does not fit 32 bits")
        heads, hd = cache.kv_heads, cache.head_dim
        if out is None:
            k = torch.empty((n_rows, heads, hd), dtype=dtype or cache.k.dtype, device=self.device)
            v = torch.empty_like(k)
            ks = vs = heads * hd
        else:
            k, v = out
            n, ks = self._heads("k", k, heads, hd)
            nv, vs = self._heads("v", v, heads, hd)
            if n < n_rows or nv < n_rows or k.dtype != v.dtype:
                _refuse("out must be two tensors of n_rows rows, alike in type")
        r = self._rows(table, cu, first)
        rc = self._L.hipvoc_kv_read(self._h, cache._p, k.data_ptr(), v.data_ptr(), ks, vs, _type(k), C.addressof(r), n_rows, self.stream)
        if rc:
            self._failed(rc)
        return k, v

    # ---- attention of one new token ------------------------------------------------------
    def attention(self, q, cache: KvCache, table, lens, scale: Optional[float] = None, window: int = 0, max_len: Optional[int] = None,
                  lse: bool = False, out=None):
        """q [seqs, heads, head_dim] over the lens[b] tokens of each sequence -> out like q; with lse=True also the log of the
        softmax's sum [seqs, heads] float32.  max_len: a bound on lens the host knows (default: all the table's pages hold)."""
        if cache.device != self.device:
            self._elsewhere("the cache", cache)
        if q.dim() != 3:
            _refuse("q must be [seqs, heads, head_dim]")
        hd, heads = cache.head_dim, q.shape[1]
        n, qs = self._heads("q", q, heads, hd)
        tp, stride, width, nt = self._table(table)
        if nt != n:
            _refuse("table must have a row per sequence")
        lp = self._ints("lens", lens, n)
        if max_len is None:
            max_len = width * cache.page
        if not (0 <= max_len < 1 << 31 and 0 <= window < 1 << 31):
            _refuse(f"max_len {max_len} or window {window} is negative or does not fit 32 bits")
        if out is None:
            out = torch.empty_like(q)
            os_ = heads * hd
        else:
            no, os_ = self._heads("out", out, heads, hd)
            if no != n or out.dtype != q.dtype:
                _refuse("out must be like q")
        sums = q.new_empty((n, heads), dtype=torch.float32) if lse else None
        need = self._L.hipvoc_attention_workspace(cache._p, heads, n, max_len, window)
        ws = lens.new_empty(need // 4) if need else None
        rc = self._L.hipvoc_attention(
            self._h, cache._p, q.data_ptr(), qs, out.data_ptr(), os_, sums.data_ptr() if lse else None, _type(q), heads, tp, stride, width, lp, n,
            max_len, window, hd ** -0.5 if scale is None else scale, ws.data_ptr() if need else None, need, self.stream)
        if rc:
            self._failed(rc)
        return (out, sums) if lse else out

    # ---- norm ----------------------------------------------------------------------------
    def add_rmsnorm(self, x, weight, residual=None, eps: float = 1e-6, quant: Optional[str] = None, group: int = 0):
        """x [rows, cols] (+ residual) -> (sum, y), or with quant "int8" / "e4m3" (sum, codes, scales [rows, cols / group]; group 0:
        one scale per row).  sum is None without a residual."""
        rows, cols, xs = self._matrix("x", x)
        act = x.dtype
        t = _type(x)
        if weight.dtype != act or weight.shape != (cols,) or not weight.is_contiguous():
            _refuse("weight must be a contiguous [cols] of x's type")
        if weight.device != self.device:
            self._elsewhere("weight", weight)
        rs, rp, total, sp = 0, None, None, None
        if residual is not None:
            rr, rc, rs = self._matrix("residual", residual)
            if residual.dtype != act or rr != rows or rc != cols:
                _refuse("residual must have x's type and shape")
            total = torch.empty_like(x)
            rp, sp = residual.data_ptr(), total.data_ptr()
        if quant is None:
            y, scales, ot, cp = torch.empty_like(x), None, t, None
        elif quant == "int8" or quant == "e4m3":
            if group and (group not in (32, 64, 128) or cols % group):
                _refuse(f"group {group} must be 0, or 32, 64 or 128 and a divisor of cols {cols}")
            ot = T_INT8 if quant == "int8" else T_E4M3
            y = torch.empty_like(x, dtype=torch.int8 if ot == T_INT8 else torch.float8_e4m3fn)
            scales = x.new_empty((rows, cols // group if group else 1), dtype=torch.float32)
            cp = scales.data_ptr()
        else:
            _refuse("quant must be None, 'int8' or 'e4m3'")
        rc = self._L.hipvoc_add_rmsnorm(self._h, x.data_ptr(), xs, rp, rs, weight.data_ptr(), sp, cols, y.data_ptr(), cols, cp, t, ot, group, eps, rows, cols,
                                        self.stream)
        if rc:
            self._failed(rc)
        return (total, y) if quant is None else (total, y, scales)

    # ---- 4-bit products ------------------------------------------------------------------
    def q4_matvec(self, codes, scales, x, mins=None, x_scale=None, dtype=None):
        """x [rows, n_in] times the 4-bit weights codes [n_out, n_in / 2] uint8, scales (mins) [n_out, n_in / group] float16 ->
        [rows, n_out].  int8 rows: x_scale [rows, n_in / group] or [rows, 1] float32, and `dtype` of the result (default float32)."""
        cs, ss = codes.shape, scales.shape
        if len(cs) != 2 or codes.dtype != torch.uint8 or not codes.is_contiguous():
            _refuse("codes must be a contiguous uint8 [n_out, n_in / 2]")
        n_out, n_in = cs[0], cs[1] * 2
        if n_out >> 31 or n_in >> 31:
            _refuse(f"codes are {n_out} rows of {n_in}")
        if len(ss) != 2 or ss[0] != n_out or scales.dtype != torch.float16 or not scales.is_contiguous() or ss[1] < 1 or n_in % ss[1]:
            _refuse("scales must be a contiguous float16 [n_out, n_in / group]")
        here, mp, xp = self.device, None, None
        if mins is not None:
            if mins.dtype != torch.float16 or mins.shape != ss or not mins.is_contiguous():
                _refuse("mins must be like scales")
            if mins.device != here:
                self._elsewhere("mins", mins)
            mp = mins.data_ptr()
        if codes.device != here or scales.device != here:
            self._elsewhere("codes or scales", codes if codes.device != here else scales)
        rows, cols, xs = self._matrix("x", x)
        if cols != n_in:
            _refuse(f"x must have {n_in} columns")
        xt, x_groups = _type(x), 0
        if xt == T_INT8:
            if x_scale is None or x_scale.dtype != torch.float32 or x_scale.dim() != 2 or x_scale.shape[0] != rows or not x_scale.is_contiguous():
                _refuse("int8 rows need x_scale, a contiguous float32 [rows, n_in / group] or [rows, 1]")
            if x_scale.device != here:
                self._elsewhere("x_scale", x_scale)
            x_groups, xp = x_scale.shape[1], x_scale.data_ptr()
            out = dtype or torch.float32
        elif x_scale is not None:
            _refuse("only int8 rows have scales")
        else:
            out = dtype or x.dtype
        y = x.new_empty((rows, n_out), dtype=out)
        rc = self._L.hipvoc_q4_matvec(self._h, codes.data_ptr(), scales.data_ptr(), mp, n_out, n_in, n_in // ss[1], x.data_ptr(), xs, xt, xp, x_groups,
                                      y.data_ptr(), n_out, _type(y), rows, self.stream)
        if rc:
            self._failed(rc)
        return y
