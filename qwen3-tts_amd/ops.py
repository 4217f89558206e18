"""ctypes binding of the token-step operators of libhipvoc.so (include/hipvoc_ops.h).

``HipOps.open(device)`` gives a handle; its methods take torch tensors of that device and enqueue on torch's current stream
of it, so they can be captured into a graph with the rest of a step.  They allocate their results (and a workspace, where one
is needed) as torch operations do; the C entry points take the caller's memory.  A refused call raises HipVocError before
anything is launched; what only the device can see (a page number, a length) is raised by ``sync()``.

There is NO fallback: if the shared library is missing or no HIP device is present, opening raises.
"""
from __future__ import annotations

import ctypes as C
import math
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


def _torch():
    import torch
    return torch


_types = {}


def _type(t) -> int:
    if not _types:
        torch = _torch()
        _types.update({torch.float32: T_F32, torch.float16: T_F16, torch.bfloat16: T_BF16, torch.int8: T_INT8, torch.float8_e4m3fn: T_E4M3})
    code = _types.get(t.dtype, -1)
    if code < 0:
        raise HipVocError(-1, f"unsupported dtype {t.dtype}")
    return code


def _refuse(msg: str):
    raise HipVocError(-1, msg)


def _int32(**values):
    """The C entry points take 32-bit integers; ctypes would wrap a larger one silently."""
    for name, v in values.items():
        if not -(1 << 31) <= v < 1 << 31:
            _refuse(f"{name} = {v} does not fit 32 bits")


class KvCache:
    """Names the tensors of a paged cache (hipvoc_kv_cache): k, v [n_pages, kv_heads, page, head_dim], contiguous within a page;
    k_scale, v_scale [n_pages, kv_heads, page] float32 for int8 / float8_e4m3fn caches."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
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
        torch = _torch()
        self._h = handle
        self._L = lib
        self.device = torch.device("cuda", device)
        self._stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None

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

    def _check(self, rc: int):
        if rc != 0:
            raise HipVocError(rc, self._L.hipvoc_last_error(self._h).decode() if self._h else "the handle is closed")

    @property
    def stream(self) -> int:
        """torch's current stream of the handle's device, where the calls are enqueued."""
        if self._stream is not None:
            return self._stream(self.device.index)
        return _torch().cuda.current_stream(self.device).cuda_stream

    def sync(self):
        """Waits for the current stream and raises what the device found wrong since the last time."""
        self._check(self._L.hipvoc_ops_sync(self._h, self.stream))

    # ---- the paged cache -----------------------------------------------------------------
    def kv_cache(self, k, v, k_scale=None, v_scale=None) -> KvCache:
        cache = KvCache(k, v, k_scale, v_scale)
        self._here(k)
        return cache

    def _here(self, *tensors):
        for t in tensors:
            if t is not None and t.device != self.device:
                _refuse(f"a tensor is on {t.device}, the handle on {self.device}")

    def _ints(self, name, t, dims):
        if t.dtype != _torch().int32 or t.dim() != dims or (t.numel() > 0 and t.stride(-1) != 1):
            _refuse(f"{name} must be int32 with {dims} dimension(s), the last contiguous")
        if t.device != self.device:
            _refuse(f"{name} is on {t.device}, the handle on {self.device}")
        return t.data_ptr()

    def _rows(self, table, cu, first):
        n = table.shape[0]
        r = _Rows(self._ints("table", table, 2), self._ints("cu", cu, 1), self._ints("first", first, 1), table.stride(0), table.shape[1], n)
        if cu.shape[0] != n + 1 or first.shape[0] != n:
            _refuse("cu must have one entry more than table has rows, first as many")
        return r

    def _heads(self, name, t, heads, hd):
        """Row stride of [rows, heads, head_dim] with contiguous rows."""
        if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != hd or (t.numel() > 0 and (t.stride(2) != 1 or (heads > 1 and t.stride(1) != hd))):
            _refuse(f"{name} must be [rows, {heads}, {hd}] with contiguous rows")
        if t.device != self.device:
            _refuse(f"{name} is on {t.device}, the handle on {self.device}")
        return t.stride(0) if t.shape[0] > 1 else heads * hd

    def kv_write(self, cache: KvCache, k, v, table, cu, first):
        """k, v [rows, kv_heads, head_dim]: rows cu[b] .. cu[b+1] go to positions first[b] ... of sequence b (pages table[b])."""
        ks, vs = self._heads("k", k, cache.kv_heads, cache.head_dim), self._heads("v", v, cache.kv_heads, cache.head_dim)
        if k.shape[0] != v.shape[0] or k.dtype != v.dtype:
            _refuse("k and v must be alike")
        self._here(cache.k)
        r = self._rows(table, cu, first)
        self._check(self._L.hipvoc_kv_write(self._h, cache._p, k.data_ptr(), v.data_ptr(), ks, vs, _type(k), C.addressof(r), k.shape[0], self.stream))

    def kv_read(self, cache: KvCache, table, cu, first, n_rows: int, dtype=None, out: Optional[Tuple] = None):
        """The inverse: (k, v) [n_rows, kv_heads, head_dim] in `dtype` (default: the cache's own), or into the two tensors of `out`;
        rows at or behind cu[-1] are left as they were."""
        torch = _torch()
        _int32(n_rows=n_rows)
        if n_rows < 0:
            _refuse(f"n_rows {n_rows} is negative")
        if out is None:
            shape = (n_rows, cache.kv_heads, cache.head_dim)
            dtype = dtype or cache.k.dtype
            out = (torch.empty(shape, dtype=dtype, device=self.device), torch.empty(shape, dtype=dtype, device=self.device))
        k, v = out
        ks, vs = self._heads("k", k, cache.kv_heads, cache.head_dim), self._heads("v", v, cache.kv_heads, cache.head_dim)
        if k.shape[0] < n_rows or v.shape[0] < n_rows or k.dtype != v.dtype:
            _refuse("out must be two tensors of n_rows rows, alike in type")
        self._here(cache.k)
        r = self._rows(table, cu, first)
        self._check(self._L.hipvoc_kv_read(self._h, cache._p, k.data_ptr(), v.data_ptr(), ks, vs, _type(k), C.addressof(r), n_rows, self.stream))
        return k, v

    # ---- attention of one new token ------------------------------------------------------
    def attention(self, q, cache: KvCache, table, lens, scale: Optional[float] = None, window: int = 0, max_len: Optional[int] = None,
                  lse: bool = False, out=None):
        """q [seqs, heads, head_dim] over the lens[b] tokens of each sequence -> out like q; with lse=True also the log of the
        softmax's sum [seqs, heads] float32.  max_len: a bound on lens the host knows (default: all the table's pages hold)."""
        torch = _torch()
        n, heads = q.shape[0], q.shape[1]
        qs = self._heads("q", q, heads, cache.head_dim)
        tp, lp = self._ints("table", table, 2), self._ints("lens", lens, 1)
        if table.shape[0] != n or lens.shape[0] != n:
            _refuse("table and lens must have a row per sequence")
        self._here(cache.k)
        width = table.shape[1]
        if max_len is None:
            max_len = width * cache.page
        _int32(window=window, max_len=max_len)
        if out is None:
            out = torch.empty((n, heads, cache.head_dim), dtype=q.dtype, device=self.device)
        os_ = self._heads("out", out, heads, cache.head_dim)
        if out.shape[0] != n or out.dtype != q.dtype:
            _refuse("out must be like q")
        sums = torch.empty((n, heads), dtype=torch.float32, device=self.device) if lse else None
        need = self._L.hipvoc_attention_workspace(cache._p, heads, n, max_len, window)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        self._check(self._L.hipvoc_attention(
            self._h, cache._p, q.data_ptr(), qs, out.data_ptr(), os_, sums.data_ptr() if lse else None, _type(q), heads, tp, table.stride(0), width, lp, n,
            max_len, window, 1.0 / math.sqrt(cache.head_dim) if scale is None else scale, ws.data_ptr() if need else None, need, self.stream))
        return (out, sums) if lse else out

    # ---- norm ----------------------------------------------------------------------------
    def _matrix(self, name, t, rows, cols):
        if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != cols or (cols > 1 and t.numel() > 0 and t.stride(1) != 1):
            _refuse(f"{name} must be [{rows}, {cols}] with contiguous rows")
        if t.device != self.device:
            _refuse(f"{name} is on {t.device}, the handle on {self.device}")
        return t.stride(0) if rows > 1 else cols

    def add_rmsnorm(self, x, weight, residual=None, eps: float = 1e-6, quant: Optional[str] = None, group: int = 0):
        """x [rows, cols] (+ residual) -> (sum, y), or with quant "int8" / "e4m3" (sum, codes, scales [rows, cols / group]; group 0:
        one scale per row).  sum is None without a residual."""
        torch = _torch()
        if x.dim() != 2:
            _refuse("x must be [rows, cols]")
        rows, cols = x.shape
        xs = self._matrix("x", x, rows, cols)
        if weight.dtype != x.dtype or weight.dim() != 1 or weight.shape[0] != cols or not weight.is_contiguous():
            _refuse("weight must be a contiguous [cols] of x's type")
        self._here(weight)
        rs, total = 0, None
        if residual is not None:
            rs = self._matrix("residual", residual, rows, cols)
            if residual.dtype != x.dtype:
                _refuse("residual must have x's type")
            total = torch.empty((rows, cols), dtype=x.dtype, device=self.device)
        if quant is None:
            y, scales, ot = torch.empty((rows, cols), dtype=x.dtype, device=self.device), None, _type(x)
        elif quant in ("int8", "e4m3"):
            _int32(group=group)
            ot = T_INT8 if quant == "int8" else T_E4M3
            y = torch.empty((rows, cols), dtype=torch.int8 if quant == "int8" else torch.float8_e4m3fn, device=self.device)
            scales = torch.empty((rows, cols // group if group > 0 else 1), dtype=torch.float32, device=self.device)
        else:
            _refuse("quant must be None, 'int8' or 'e4m3'")
        self._check(self._L.hipvoc_add_rmsnorm(
            self._h, x.data_ptr(), xs, None if residual is None else residual.data_ptr(), rs, weight.data_ptr(), None if total is None else total.data_ptr(),
            cols, y.data_ptr(), cols, None if scales is None else scales.data_ptr(), _type(x), ot, group, eps, rows, cols, self.stream))
        return (total, y) if quant is None else (total, y, scales)

    # ---- 4-bit products ------------------------------------------------------------------
    def q4_matvec(self, codes, scales, x, mins=None, x_scale=None, dtype=None):
        """x [rows, n_in] times the 4-bit weights codes [n_out, n_in / 2] uint8, scales (mins) [n_out, n_in / group] float16 ->
        [rows, n_out].  int8 rows: x_scale [rows, n_in / group] or [rows, 1] float32, and `dtype` of the result (default float32)."""
        torch = _torch()
        if codes.dim() != 2 or codes.dtype != torch.uint8 or not codes.is_contiguous() or scales.dim() != 2 or x.dim() != 2:
            _refuse("codes must be a contiguous uint8 [n_out, n_in / 2], scales [n_out, n_in / group], x [rows, n_in]")
        n_out, n_in, rows = codes.shape[0], codes.shape[1] * 2, x.shape[0]
        groups = scales.shape[1]
        for t in (scales, mins):
            if t is not None and (t.dtype != torch.float16 or tuple(t.shape) != (n_out, groups) or not t.is_contiguous()):
                _refuse("scales and mins must be contiguous float16 [n_out, n_in / group]")
        if groups < 1 or n_in % groups:
            _refuse("scales must have a column per group of n_in")
        self._here(codes, scales, mins, x_scale)
        xs = self._matrix("x", x, rows, n_in)
        xt, x_groups = _type(x), 0
        if xt == T_INT8:
            if x_scale is None or x_scale.dtype != torch.float32 or x_scale.dim() != 2 or x_scale.shape[0] != rows or not x_scale.is_contiguous():
                _refuse("int8 rows need x_scale, a contiguous float32 [rows, n_in / group] or [rows, 1]")
            x_groups = x_scale.shape[1]
        elif x_scale is not None:
            _refuse("only int8 rows have scales")
        y = torch.empty((rows, n_out), dtype=dtype or (torch.float32 if xt == T_INT8 else x.dtype), device=self.device)
        self._check(self._L.hipvoc_q4_matvec(
            self._h, codes.data_ptr(), scales.data_ptr(), None if mins is None else mins.data_ptr(), n_out, n_in, n_in // groups, x.data_ptr(), xs, xt,
            None if x_scale is None else x_scale.data_ptr(), x_groups, y.data_ptr(), n_out, _type(y), rows, self.stream))
        return y
