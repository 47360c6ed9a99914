"""torch view of the paged key/value cache operators (include/mocha_kv.h).

    cache = KvPages(k, v)          # [pages, kv heads, page size, head dim], any strides of the first three
    q = cache.append(q, k_new, v_new, seq, pos, table, cos=cos, sin=sin)
    out = cache.decode(q, table, kv_len)                # one new token per sequence
    out = cache.prefill(q, q_start, table, kv_len)      # ragged prompt pieces

The calls enqueue on torch's current stream of the pages' device and can be captured into
CUDA graphs; outputs and workspaces that the caller does not pass come from torch's
allocator, call by call.  Arguments that do not fit raise ValueError before anything is
enqueued; an error from the library raises RuntimeError.  There are no gradients: a tensor
that requires one is refused unless gradients are off, and so is one with a tangent of
forward mode.  No reference counterpart.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd import forward_ad

import mocha_native

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class _Pages(C.Structure):
    _fields_ = [("device", C.c_int), ("type", C.c_int), ("pages", C.c_int), ("page_size", C.c_int),
                ("kv_heads", C.c_int), ("head_dim", C.c_int), ("page_stride", C.c_longlong),
                ("head_stride", C.c_longlong), ("token_stride", C.c_longlong), ("k", C.c_void_p), ("v", C.c_void_p)]


class _Seqs(C.Structure):
    _fields_ = [("seqs", C.c_int), ("table_width", C.c_int), ("table_stride", C.c_longlong), ("table", C.c_void_p),
                ("kv_len", C.c_void_p), ("status", C.c_void_p)]


class _Rows(C.Structure):
    _fields_ = [("data", C.c_void_p), ("row_stride", C.c_longlong), ("head_stride", C.c_longlong)]


class _Rope(C.Structure):
    _fields_ = [("cos", C.c_void_p), ("sin", C.c_void_p), ("stride", C.c_longlong), ("positions", C.c_int),
                ("dims", C.c_int), ("interleaved", C.c_int)]


class _Scores(C.Structure):
    _fields_ = [("heads", C.c_int), ("window", C.c_int), ("scale", C.c_float), ("cap", C.c_float),
                ("prefix", C.c_void_p), ("slopes", C.c_void_p)]


_SIGS = {
    "mocha_kv_append": [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p,
                        C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p],
    "mocha_kv_workspace": [C.c_void_p, C.c_int, C.c_int, C.c_void_p],
    "mocha_kv_decode": [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                        C.c_ulonglong, C.c_void_p],
    "mocha_kv_prefill": [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                         C.c_void_p, C.c_ulonglong, C.c_void_p],
    "mocha_kv_prefill_check": [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p,
                               C.c_void_p, C.c_void_p, C.c_ulonglong, C.c_void_p, C.c_int, C.c_int],
}

_lib = None


def _no_gradient(names, *tensors):
    if forward_ad._current_level < 0:
        for t in tensors:
            if t is not None and t.requires_grad:
                break
        else:
            return
    for name, t in zip(names.split(), tensors):
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient, which these operators do not have")
        if t is not None and forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{name} has a tangent, which these operators do not carry on")


def _load() -> C.CDLL:
    global _lib
    if _lib is None:
        lib = mocha_native.load()
        for name, args in _SIGS.items():
            fn = getattr(lib, name)
            fn.restype = C.c_int
            fn.argtypes = args
        _lib = lib
    return _lib


_stream = torch._C._cuda_getCurrentRawStream  # current_stream(device).cuda_stream in 0.1 us in place of 1.3


class KvPages:
    """A page pool on one device: k and v, [pages, kv_heads, page_size, head_dim] tensors (or
    views) of one type, fp32, fp16 or bf16, with the same strides."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if k.dim() != 4 or k.shape != v.shape:
            raise ValueError("k and v must be [pages, kv_heads, page_size, head_dim]")
        if k.dtype not in _TYPES or k.dtype != v.dtype:
            raise ValueError("k and v must be float32, float16 or bfloat16, of one type")
        if k.stride() != v.stride() or k.stride(3) != 1:
            raise ValueError("k and v must have the same strides, the last one 1")
        _no_gradient("k v", k, v)
        if k.device.type != "cuda" or k.device != v.device:
            raise ValueError("k and v must be on one CUDA device")
        self.k, self.v = k, v
        self.device, self.dtype = k.device, k.dtype
        self.kv_heads, self.page_size, self.head_dim = k.shape[1:]
        self._index = k.get_device()
        self._p = _Pages(self._index, _TYPES[k.dtype], k.shape[0], k.shape[2], k.shape[1], k.shape[3], k.stride(0),
                         k.stride(1), k.stride(2), k.data_ptr(), v.data_ptr())
        self._pages = C.addressof(self._p)
        self._bytes = {}

    # -- argument views (messages are put together only when a check fails) --------------

    def _int(self, t, name, n):
        if t.dtype is not torch.int32 or t.get_device() != self._index or t.shape != (n,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 vector of {n} on the pages' device")
        return t.data_ptr()

    def _seqs(self, table, kv_len, status):
        shape = table.shape
        if (len(shape) != 2 or table.dtype is not torch.int32 or table.get_device() != self._index or
                (shape[1] > 1 and table.stride(1) != 1)):
            raise ValueError("table must be an int32 matrix [seqs, pages of a sequence] on the pages' device")
        n, width = shape
        return _Seqs(n, width, table.stride(0) if n > 1 else width, table.data_ptr(),
                     None if kv_len is None else self._int(kv_len, "kv_len", n),
                     None if status is None else self._int(status, "status", 1))

    def _rows(self, t, name, dtype, rows, heads=None):
        shape = t.shape
        if (len(shape) != 3 or t.dtype is not dtype or t.get_device() != self._index or shape[0] != rows or
                shape[2] != self.head_dim or (heads is not None and shape[1] != heads)):
            raise ValueError(f"{name} must be [{rows}, {heads or 'heads'}, {self.head_dim}] of {dtype} on the pages' device")
        row, head, one = t.stride()
        if one != 1:
            raise ValueError(f"{name}: a head's values must be contiguous")
        return _Rows(t.data_ptr(), row if rows > 1 else 0, head if shape[1] > 1 else self.head_dim)

    def _scores(self, heads, n, scale, window, prefix, cap, slopes):
        if slopes is not None:
            if (slopes.dtype is not torch.float32 or slopes.get_device() != self._index or slopes.shape != (heads,) or
                    not slopes.is_contiguous()):
                raise ValueError(f"slopes must be a contiguous float32 vector of {heads} on the pages' device")
            slopes = slopes.data_ptr()
        if not 0 <= window < 1 << 31:  # ctypes would keep the low 32 bits
            window = -1 if window < 0 else (1 << 31) - 1
        return _Scores(heads, window, self.head_dim ** -0.5 if scale is None else scale, cap,
                       None if prefix is None else self._int(prefix, "prefix", n), slopes)

    def _lse(self, lse, rows, heads):
        if lse is None:
            return None
        if (lse.dtype is not torch.float32 or lse.get_device() != self._index or lse.shape != (rows, heads) or
                not lse.is_contiguous()):
            raise ValueError(f"lse must be a contiguous float32 [{rows}, {heads}] on the pages' device")
        return lse.data_ptr()

    def _space(self, lib, heads, prefill):
        n = self._bytes.get((heads, prefill))
        if n is None:
            got = C.c_ulonglong()
            if lib.mocha_kv_workspace(self._pages, heads, prefill, C.byref(got)):
                raise RuntimeError("mocha_kv_workspace failed")
            n = self._bytes[heads, prefill] = got.value
        return n, torch.empty(n, dtype=torch.uint8, device=self.device)

    # -- operators ----------------------------------------------------------------------

    def append(self, q, k, v, seq, pos, table, *, cos=None, sin=None, interleaved=False, q_out=None, status=None):
        """Rotary positions on q [rows, heads, dim] (or None) and k [rows, kv_heads, dim], and k
        and v into the pages of (seq[i], pos[i]); rows with a negative seq are skipped.  cos and
        sin: [positions, rotated dims / 2] float32, or None for no rotation.  Returns q_out."""
        lib = _lib or _load()
        rows = k.shape[0]
        if k.dtype not in _TYPES:
            raise ValueError("k must be float32, float16 or bfloat16")
        kr = self._rows(k, "k", k.dtype, rows, self.kv_heads)
        vr = self._rows(v, "v", k.dtype, rows, self.kv_heads)
        qr = orr = None
        heads = 0
        if q is not None:
            qr = self._rows(q, "q", k.dtype, rows)
            heads = q.shape[1]
            if q_out is None:
                q_out = torch.empty(rows, heads, self.head_dim, dtype=self.dtype, device=self.device)
            orr = self._rows(q_out, "q_out", self.dtype, rows, heads)
        elif q_out is not None:
            raise ValueError("q_out without q")
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin go together")
        if cos is None:
            rope = _Rope(None, None, 0, 0, 0, 0)
        else:
            if (cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or cos.dim() != 2 or
                    cos.shape != sin.shape or cos.get_device() != self._index or sin.get_device() != self._index or
                    cos.stride() != sin.stride() or cos.stride(1) != 1):
                raise ValueError("cos and sin must be float32 [positions, rotated dims / 2] with the same strides on "
                                 "the pages' device")
            rope = _Rope(cos.data_ptr(), sin.data_ptr(), cos.stride(0) if cos.shape[0] > 1 else cos.shape[1], cos.shape[0],
                         2 * cos.shape[1],
                         int(bool(interleaved)))
        seqs = self._seqs(table, None, status)
        _no_gradient("q k v q_out cos sin pages.k pages.v", q, k, v, q_out, cos, sin, self.k, self.v)
        if lib.mocha_kv_append(self._pages, C.addressof(seqs), rows, self._int(seq, "seq", rows),
                               self._int(pos, "pos", rows), _TYPES[k.dtype], heads, qr and C.addressof(qr),
                               C.addressof(kr), C.addressof(vr), orr and C.addressof(orr), C.addressof(rope),
                               _stream(self._index)):
            raise RuntimeError("mocha_kv_append failed")
        return q_out

    def decode(self, q, table, kv_len, *, scale=None, window=0, prefix=None, cap=0.0, slopes=None, out=None, lse=None,
               status=None):
        """Attention of q [seqs, heads, dim], the sequences' last positions; scale defaults to
        dim ** -0.5.  Returns out."""
        lib = _lib or _load()
        n = table.shape[0]
        qr = self._rows(q, "q", self.dtype, n)
        heads = q.shape[1]
        if out is None:
            out = torch.empty(n, heads, self.head_dim, dtype=self.dtype, device=self.device)
        orr = self._rows(out, "out", self.dtype, n, heads)
        seqs = self._seqs(table, kv_len, status)
        scores = self._scores(heads, n, scale, window, prefix, cap, slopes)
        _no_gradient("q slopes out lse pages.k pages.v", q, slopes, out, lse, self.k, self.v)
        size, space = self._space(lib, heads, 0)
        if lib.mocha_kv_decode(self._pages, C.addressof(seqs), C.addressof(scores), C.addressof(qr), C.addressof(orr),
                               self._lse(lse, n, heads), space.data_ptr(), size,
                               _stream(self._index)):
            raise RuntimeError("mocha_kv_decode failed")
        return out

    def prefill(self, q, q_start, table, kv_len, *, scale=None, window=0, prefix=None, cap=0.0, slopes=None, out=None,
                lse=None, status=None):
        """Attention of q [rows, heads, dim], rows q_start[s] .. q_start[s + 1] - 1 being the last
        positions of sequence s.  Rows outside every range are left as they were.  Returns out."""
        lib = _lib or _load()
        rows, n = q.shape[0], table.shape[0]
        qr = self._rows(q, "q", self.dtype, rows)
        heads = q.shape[1]
        if out is None:
            out = torch.empty(rows, heads, self.head_dim, dtype=self.dtype, device=self.device)
        orr = self._rows(out, "out", self.dtype, rows, heads)
        seqs = self._seqs(table, kv_len, status)
        scores = self._scores(heads, n, scale, window, prefix, cap, slopes)
        _no_gradient("q slopes out lse pages.k pages.v", q, slopes, out, lse, self.k, self.v)
        size, space = self._space(lib, heads, 1)
        if lib.mocha_kv_prefill(self._pages, C.addressof(seqs), C.addressof(scores), rows,
                                self._int(q_start, "q_start", n + 1), C.addressof(qr), C.addressof(orr),
                                self._lse(lse, rows, heads), space.data_ptr(), size,
                                _stream(self._index)):
            raise RuntimeError("mocha_kv_prefill failed")
        return out
