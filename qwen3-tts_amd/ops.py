"""The token-step operators of libhipvoc.so (include/hipvoc_ops.h) on torch tensors.

``HipOps.open(device)`` gives a handle; its methods take torch tensors of that device and enqueue on torch's current stream
of it, so they can be captured into a graph with the rest of a step.  They allocate their results (and a workspace, where one
is needed) as torch operations do; the C entry points take the caller's memory.  A refused call raises HipVocError before
anything is launched; what only the device can see (a page number, a length) is raised by ``sync()``.
They are for inference: there is no backward pass, and while gradients are recorded a tensor that requires one is refused.

The tensors are looked at in _ops_torch.so (csrc/ops_torch.cpp), which calls the C entry points; here they have their names.
There is NO fallback: if a shared library is missing or no HIP device is present, opening raises.
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


# The C entry points for a caller that holds addresses, not tensors: their structs, and in _lib() their arguments.
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
_native = None                  # _ops_torch.so
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
    k_scale, v_scale [n_pages, kv_heads, page] float32 for int8 / float8_e4m3fn caches.  None of them requires a gradient."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        _bind_torch()
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            _refuse("k and v must be [n_pages, kv_heads, page, head_dim], alike in shape, type and device")
        n, heads, page, hd = k.shape
        for t in (k, v, k_scale, v_scale):
            if t is not None and (t.requires_grad or t.is_neg()):
                _refuse("a cache's tensors carry no gradient (detach them) and are no views of a negative (resolve_neg)")
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


def _bind_native():
    global _native
    if _native is None:
        _bind_torch()
        from . import _ops_torch as module
        L = _lib()
        at = lambda name: C.cast(getattr(L, name), C.c_void_p).value  # noqa: E731
        module.bind(HipVocError, *[at("hipvoc_" + n) for n in ("kv_write", "kv_read", "attention_workspace", "attention", "add_rmsnorm", "q4_matvec", "last_error")])
        _native = module


class HipOps:
    """The operators of one token step on one MI355X."""

    def __init__(self, handle, lib, device: int):
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
        try:
            _bind_native()
        except BaseException:
            L.hipvoc_free(h)
            raise
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

    @property
    def stream(self) -> int:
        """torch's current stream of the handle's device, where the calls are enqueued."""
        return torch._C._cuda_getCurrentRawStream(self._index)

    def sync(self):
        """Waits for the current stream and raises what the device found wrong since the last time, in calls of any stream on this handle."""
        rc = self._L.hipvoc_ops_sync(self._h, self.stream)
        if rc:
            raise HipVocError(rc, self._L.hipvoc_last_error(self._h).decode() if self._h else "the handle is closed")

    # ---- the paged cache -----------------------------------------------------------------
    def kv_cache(self, k, v, k_scale=None, v_scale=None) -> KvCache:
        if k.device != self.device:
            _refuse(f"k is on {k.device}, the handle on {self.device}")
        return KvCache(k, v, k_scale, v_scale)

    def kv_write(self, cache: KvCache, k, v, table, cu, first):
        """k, v [rows, kv_heads, head_dim]: rows cu[b] .. cu[b+1] go to positions first[b] ... of sequence b (pages table[b])."""
        _native.kv_write(self._h, self._index, cache, k, v, table, cu, first)

    def kv_read(self, cache: KvCache, table, cu, first, n_rows: int, dtype=None, out: Optional[Tuple] = None):
        """The inverse: (k, v) [n_rows, kv_heads, head_dim] in `dtype` (default: the cache's own), or into the two tensors of `out`;
        rows at or behind cu[-1] are left as they were."""
        return _native.kv_read(self._h, self._index, cache, table, cu, first, n_rows, dtype, out)

    # ---- attention of one new token ------------------------------------------------------
    def attention(self, q, cache: KvCache, table, lens, scale: Optional[float] = None, window: int = 0, max_len: Optional[int] = None,
                  lse: bool = False, out=None):
        """q [seqs, heads, head_dim] over the lens[b] tokens of each sequence -> out like q; with lse=True also the log of the
        softmax's sum [seqs, heads] float32.  max_len: a bound on lens the host knows (default: all the table's pages hold)."""
        return _native.attention(self._h, self._index, q, cache, table, lens, scale, window, max_len, lse, out)

    # ---- norm ----------------------------------------------------------------------------
    def add_rmsnorm(self, x, weight, residual=None, eps: float = 1e-6, quant: Optional[str] = None, group: int = 0):
        """x [rows, cols] (+ residual) -> (sum, y), or with quant "int8" / "e4m3" (sum, codes, scales [rows, cols / group]; group 0:
        one scale per row).  sum is None without a residual."""
        if quant is not None:
            quant = T_INT8 if quant == "int8" else T_E4M3 if quant == "e4m3" else _refuse("quant must be None, 'int8' or 'e4m3'")
        return _native.add_rmsnorm(self._h, self._index, x, weight, residual, eps, quant, group)

    # ---- 4-bit products ------------------------------------------------------------------
    def q4_matvec(self, codes, scales, x, mins=None, x_scale=None, dtype=None):
        """x [rows, n_in] times the 4-bit weights codes [n_out, n_in / 2] uint8, scales (mins) [n_out, n_in / group] float16 ->
        [rows, n_out].  int8 rows: x_scale [rows, n_in / group] or [rows, 1] float32, and `dtype` of the result (default float32)."""
        return _native.q4_matvec(self._h, self._index, codes, scales, x, mins, x_scale, dtype)
