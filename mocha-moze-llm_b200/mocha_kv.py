"""torch view of the paged key/value cache operators (include/mocha_kv.h).

    cache = KvPages(k, v)          # [pages, kv heads, page size, head dim], any strides of the first three
    q = cache.append(q, k_new, v_new, seq, pos, table, cos=cos, sin=sin)
    out = cache.decode(q, table, kv_len)                # one new token per sequence
    out = cache.prefill(q, q_start, table, kv_len)      # ragged prompt pieces

The calls enqueue on torch's current stream of the pages' device and can be captured into
CUDA graphs; outputs and workspaces that the caller does not pass come from torch's
allocator, call by call.  Arguments that do not fit raise ValueError before anything is
enqueued; an error from the library raises RuntimeError.  No reference counterpart.
"""
from __future__ import annotations

import ctypes as C

import torch

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
}

_lib = None


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


def _need(ok: bool, what: str):
    if not ok:
        raise ValueError(what)


class KvPages:
    """A page pool on one device: k and v, [pages, kv_heads, page_size, head_dim] tensors (or
    views) of one type, fp32, fp16 or bf16, with the same strides."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        _need(k.dim() == 4 and k.shape == v.shape, "k and v must be [pages, kv_heads, page_size, head_dim]")
        _need(k.dtype in _TYPES and k.dtype == v.dtype, "k and v must be float32, float16 or bfloat16, of one type")
        _need(k.stride() == v.stride() and k.stride(3) == 1, "k and v must have the same strides, the last one 1")
        _need(k.device.type == "cuda" and k.device == v.device, "k and v must be on one CUDA device")
        self.k, self.v = k, v
        self.device, self.dtype = k.device, k.dtype
        self.kv_heads, self.page_size, self.head_dim = k.shape[1:]
        self._p = _Pages(k.device.index, _TYPES[k.dtype], k.shape[0], k.shape[2], k.shape[1], k.shape[3], k.stride(0),
                         k.stride(1), k.stride(2), k.data_ptr(), v.data_ptr())
        self._pages = C.addressof(self._p)
        self._bytes = {}

    # -- argument views -----------------------------------------------------------------

    def _int(self, t, name, n=None):
        _need(t.dtype == torch.int32 and t.device == self.device and t.dim() == 1 and t.is_contiguous() and
              (n is None or t.shape[0] == n),
              f"{name} must be a contiguous int32 vector on the pages' device" + (f" of {n}" if n is not None else ""))
        return t.data_ptr()

    def _seqs(self, table, kv_len, status):
        _need(table.dim() == 2 and table.dtype == torch.int32 and table.device == self.device and
              (table.shape[1] < 2 or table.stride(1) == 1),
              "table must be an int32 matrix [seqs, pages of a sequence] on the pages' device")
        n, width = table.shape
        return _Seqs(n, width, max(table.stride(0), width) if n < 2 else table.stride(0), table.data_ptr(),
                     None if kv_len is None else self._int(kv_len, "kv_len", n),
                     None if status is None else self._int(status, "status", 1))

    def _rows(self, t, name, dtype, rows, heads=None):
        _need(t.dim() == 3 and t.dtype == dtype and t.device == self.device and t.shape[0] == rows and
              t.shape[2] == self.head_dim and t.stride(2) == 1 and (heads is None or t.shape[1] == heads),
              f"{name} must be [{rows}, {heads or 'heads'}, {self.head_dim}] of {dtype} on the pages' device, "
              "a head's values contiguous")
        return _Rows(t.data_ptr(), t.stride(0) if rows > 1 else 0, t.stride(1) if t.shape[1] > 1 else self.head_dim)

    def _scores(self, heads, n, scale, window, prefix, cap, slopes):
        if slopes is not None:
            _need(slopes.dtype == torch.float32 and slopes.device == self.device and slopes.is_contiguous() and
                  slopes.shape == (heads,), f"slopes must be a contiguous float32 vector of {heads} on the pages' device")
            slopes = slopes.data_ptr()
        return _Scores(heads, window, self.head_dim ** -0.5 if scale is None else scale, cap,
                       None if prefix is None else self._int(prefix, "prefix", n), slopes)

    def _lse(self, lse, rows, heads):
        if lse is None:
            return None
        _need(lse.dtype == torch.float32 and lse.device == self.device and lse.is_contiguous() and
              lse.shape == (rows, heads), f"lse must be a contiguous float32 [{rows}, {heads}] on the pages' device")
        return lse.data_ptr()

    def _space(self, lib, heads, prefill):
        n = self._bytes.get((heads, prefill))
        if n is None:
            got = C.c_ulonglong()
            if lib.mocha_kv_workspace(self._pages, heads, prefill, C.byref(got)):
                raise RuntimeError("mocha_kv_workspace failed")
            n = self._bytes[heads, prefill] = got.value
        return torch.empty(n, dtype=torch.uint8, device=self.device)

    # -- operators ----------------------------------------------------------------------

    def append(self, q, k, v, seq, pos, table, *, cos=None, sin=None, interleaved=False, q_out=None, status=None):
        """Rotary positions on q [rows, heads, dim] (or None) and k [rows, kv_heads, dim], and k
        and v into the pages of (seq[i], pos[i]); rows with a negative seq are skipped.  cos and
        sin: [positions, rotated dims / 2] float32, or None for no rotation.  Returns q_out."""
        lib = _load()
        rows = k.shape[0]
        _need(k.dtype in _TYPES, "k must be float32, float16 or bfloat16")
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
        else:
            _need(q_out is None, "q_out without q")
        _need((cos is None) == (sin is None), "cos and sin go together")
        if cos is None:
            rope = _Rope(None, None, 0, 0, 0, 0)
        else:
            _need(cos.dtype == torch.float32 and sin.dtype == torch.float32 and cos.dim() == 2 and
                  cos.shape == sin.shape and cos.device == self.device and sin.device == self.device and
                  cos.stride(1) == 1 and cos.stride() == sin.stride(),
                  "cos and sin must be float32 [positions, rotated dims / 2] with the same strides on the pages' device")
            rope = _Rope(cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.shape[0], 2 * cos.shape[1],
                         int(bool(interleaved)))
        seqs = self._seqs(table, None, status)
        if lib.mocha_kv_append(self._pages, C.addressof(seqs), rows, self._int(seq, "seq", rows),
                               self._int(pos, "pos", rows), _TYPES[k.dtype], heads, qr and C.addressof(qr),
                               C.addressof(kr), C.addressof(vr), orr and C.addressof(orr), C.addressof(rope),
                               torch.cuda.current_stream(self.device).cuda_stream):
            raise RuntimeError("mocha_kv_append failed")
        return q_out

    def decode(self, q, table, kv_len, *, scale=None, window=0, prefix=None, cap=0.0, slopes=None, out=None, lse=None,
               status=None):
        """Attention of q [seqs, heads, dim], the sequences' last positions; scale defaults to
        dim ** -0.5.  Returns out."""
        lib = _load()
        n = table.shape[0]
        qr = self._rows(q, "q", self.dtype, n)
        heads = q.shape[1]
        if out is None:
            out = torch.empty(n, heads, self.head_dim, dtype=self.dtype, device=self.device)
        orr = self._rows(out, "out", self.dtype, n, heads)
        seqs = self._seqs(table, kv_len, status)
        scores = self._scores(heads, n, scale, window, prefix, cap, slopes)
        space = self._space(lib, heads, 0)
        if lib.mocha_kv_decode(self._pages, C.addressof(seqs), C.addressof(scores), C.addressof(qr), C.addressof(orr),
                               self._lse(lse, n, heads), space.data_ptr(), space.numel(),
                               torch.cuda.current_stream(self.device).cuda_stream):
            raise RuntimeError("mocha_kv_decode failed")
        return out

    def prefill(self, q, q_start, table, kv_len, *, scale=None, window=0, prefix=None, cap=0.0, slopes=None, out=None,
                lse=None, status=None):
        """Attention of q [rows, heads, dim], rows q_start[s] .. q_start[s + 1] - 1 being the last
        positions of sequence s.  Rows outside every range are left as they were.  Returns out."""
        lib = _load()
        rows, n = q.shape[0], table.shape[0]
        qr = self._rows(q, "q", self.dtype, rows)
        heads = q.shape[1]
        if out is None:
            out = torch.empty(rows, heads, self.head_dim, dtype=self.dtype, device=self.device)
        orr = self._rows(out, "out", self.dtype, rows, heads)
        seqs = self._seqs(table, kv_len, status)
        scores = self._scores(heads, n, scale, window, prefix, cap, slopes)
        space = self._space(lib, heads, 1)
        if lib.mocha_kv_prefill(self._pages, C.addressof(seqs), C.addressof(scores), rows,
                                self._int(q_start, "q_start", n + 1), C.addressof(qr), C.addressof(orr),
                                self._lse(lse, rows, heads), space.data_ptr(), space.numel(),
                                torch.cuda.current_stream(self.device).cuda_stream):
            raise RuntimeError("mocha_kv_prefill failed")
        return out
