"""The paged key/value cache (cpg_kv_* of include/cpg.h): append rows, attend over what is cached.

    cache = KVCache(k_pool, v_pool, rope_dim=128, rope_theta=1e6)
    batch = KVBatch(q_start, pos0, pages, rows=T, max_new=most)
    q = cache.append(batch, q, k, v, q_norm=gq, k_norm=gk)
    out = cache.attend(batch, q, ws=cache.workspace(n_heads))

The reference keeps one contiguous f32 cache per sequence (engine/blocks/qwen3_moe.h:40-70); here
sequences of any length share pools of pages. Device memory is torch CUDA tensors; every computation
runs in libcpg_b200.so.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import KvDesc, KvRows, check, lib

_TYPES = {torch.float32: _lib.T_F32, torch.float16: _lib.T_F16, torch.bfloat16: _lib.T_BF16}


_ALL = 2 ** 31 - 1                                       # a window past every position (and the C entry's int)


def _require(ok: bool, msg: str) -> None:
    if not ok:
        raise _lib.CpgError(_lib.CPG_EINVAL, msg)


def _ints(t, what: str, ndim: int, device):
    _require(isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.dim() == ndim and t.device == device
             and (t.numel() == 0 or t.stride(-1) == 1 or t.shape[-1] == 1),
             f"{what} must be an int32 tensor of {ndim} dimension(s) on {device}, its last one dense")
    return t


class KVBatch:
    """The rows of a step: sequence i brings rows q_start[i] .. q_start[i+1]-1, the first of them at
    position pos0[i], its positions in the pages of table row i. The tensors are kept and read when
    the kernels run: change them in place between steps, or replay a captured step after that. Rows of
    no sequence are not written. max_new: the most rows a sequence brings (0: not known), which chooses
    the kernel: give 1 for a step of single tokens."""

    def __init__(self, q_start, pos0, pages, *, rows: int, max_new: int = 0):
        _require(isinstance(q_start, torch.Tensor) and q_start.is_cuda, "q_start must be a CUDA tensor")
        dev = q_start.device
        self.q_start, self.pos0 = _ints(q_start, "q_start", 1, dev), _ints(pos0, "pos0", 1, dev)
        self.pages = _ints(pages, "pages", 2, dev)
        n = pos0.shape[0]
        _require(q_start.shape[0] == n + 1 and pages.shape[0] == n,
                 f"{n} sequences need {n + 1} starts and {n} table rows, got {q_start.shape[0]} and {pages.shape[0]}")
        _require(rows >= 0 and max_new >= 0, "rows and max_new must not be negative")
        self.device, self.index, self.n_seqs, self.rows = dev, q_start.get_device(), n, int(rows)
        wide = pages.shape[1]
        stride = pages.stride(0) if n > 1 else wide
        self._c = KvRows(n, self.rows, q_start.data_ptr(), pos0.data_ptr(), pages.data_ptr(), stride, wide, int(max_new))
        self._ref = ctypes.byref(self._c)


class KVCache:
    """Key and value pools (n_pages, page_size, n_kv, head_dim), f32, f16 or bf16, in any memory order
    whose last axis is dense (a pool stored head by head: pool.transpose(1, 2)). Queries and keys
    are rotated over their first rope_dim elements (None: all of them, 0: none); rope_f32 takes the
    reference's f32 angles (engine/kernels/kernels.c:425-447) instead of exact ones. For inference:
    results carry no gradient, whatever the inputs ask for."""

    def __init__(self, k_pool, v_pool, *, rope_dim: int | None = None, rope_theta: float = 1e6, rope_f32: bool = False):
        for name, p in (("k_pool", k_pool), ("v_pool", v_pool)):
            _require(isinstance(p, torch.Tensor) and p.is_cuda and p.dim() == 4 and p.dtype in _TYPES and p.numel() > 0,
                     f"{name} must be a CUDA tensor (n_pages, page_size, n_kv, head_dim) of f32, f16 or bf16")
            _require(p.stride(3) == 1, f"{name}: the last axis must be dense")
        _require(k_pool.shape == v_pool.shape and k_pool.dtype == v_pool.dtype and k_pool.device == v_pool.device
                 and all(n == 1 or a == b for n, a, b in zip(k_pool.shape, k_pool.stride(), v_pool.stride())),
                 "k_pool and v_pool must agree in shape, strides, type and device")
        self.k_pool, self.v_pool, self.device = k_pool, v_pool, k_pool.device
        self._index = k_pool.get_device()
        self.n_pages, self.page_size, self.n_kv, self.head_dim = k_pool.shape
        self.dtype, self._type = k_pool.dtype, _TYPES[k_pool.dtype]
        sp, st, sh, _ = k_pool.stride()
        desc = KvDesc(self.n_kv, self.head_dim, self.page_size, self.n_pages, self._type, k_pool.data_ptr(),
                      v_pool.data_ptr(), sp, st, sh, self.head_dim if rope_dim is None else int(rope_dim),
                      rope_theta, 1 if rope_f32 else 0)
        self._scale = self.head_dim ** -0.5
        h = ctypes.c_void_p()
        with torch.cuda.device(self.device):
            check(lib().cpg_kv_create(ctypes.byref(desc), ctypes.byref(h)))
        self.handle = h
        self._append, self._attend = lib().cpg_kv_append, lib().cpg_kv_attend

    def workspace(self, n_heads: int, stream=None):
        """A workspace of attend(), for any batch of n_heads query heads; overlapping calls need one
        each. Zeroed on `stream` (default: the current one)."""
        n = int(lib().cpg_kv_attend_workspace_bytes(self.handle, int(n_heads)))
        _require(n > 0, _lib.last_error())
        with torch.cuda.stream(stream):
            return torch.zeros(n, dtype=torch.uint8, device=self.device)

    def _rows(self, t, what: str, rows: int, heads: int | None):
        """Row stride of t (rows, heads, head_dim) after its checks."""
        shape, stride, hd = t.shape, t.stride(), self.head_dim
        if len(shape) == 3 and shape[0] == rows and shape[2] == hd and stride[2] == 1 and (
                shape[1] == heads or heads is None) and (stride[1] == hd or shape[1] == 1) and (
                t.get_device() == self._index and t.dtype in _TYPES):
            return stride[0] if rows > 1 else shape[1] * hd
        raise _lib.CpgError(_lib.CPG_EINVAL, f"{what} of shape {tuple(shape)}, strides {stride}, {t.dtype} on {t.device}: "
                            f"({rows}, {'heads' if heads is None else heads}, {hd}) of f32 or the cache's type, the heads "
                            f"of a row dense, on {self.device}")

    def _call(self, stream, fn, *args):
        index = self._index
        if torch._C._cuda_getDevice() != index:
            with torch.cuda.device(index):
                return self._call(stream, fn, *args)
        s = stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(index)
        rc = fn(self.handle, *args, s)
        if rc:
            check(rc)

    def append(self, batch: KVBatch, q, k, v, *, q_norm=None, k_norm=None, eps: float = 1e-6, q_out=None, stream=None):
        """Keys and values of the batch's rows into their pages; returns the queries, normed and
        rotated like the keys (q_out: written there; may be q). q (rows, n_heads, head_dim) or None,
        k and v (rows, n_kv, head_dim); q_norm, k_norm f32 gains (head_dim) or None."""
        _require(batch.index == self._index, "the batch and the cache must be on one device")
        ks, vs = self._rows(k, "k", batch.rows, self.n_kv), self._rows(v, "v", batch.rows, self.n_kv)
        dt = k.dtype
        heads = qs = os_ = 0
        if q is not None:
            qs, heads = self._rows(q, "q", batch.rows, None), q.shape[1]
            if q_out is None:
                with torch.cuda.stream(stream):          # memory that is free on the stream that writes it
                    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            os_ = self._rows(q_out, "q_out", batch.rows, heads)
            _require(q.dtype == dt and q_out.dtype == dt, "q, k, v and q_out must have one type")
        else:
            _require(q_out is None, "q_out without q")
        _require(v.dtype == dt, "q, k, v and q_out must have one type")
        for g in (q_norm, k_norm):
            _require(g is None or (g.dtype is torch.float32 and g.shape == (self.head_dim,) and g.is_contiguous()
                                   and g.get_device() == self._index), "gains are f32 (head_dim) on the cache's device")
        self._call(stream, self._append, batch._ref, _TYPES[dt], heads, None if q is None else q.data_ptr(), qs,
                   k.data_ptr(), ks, v.data_ptr(), vs, None if q_norm is None else q_norm.data_ptr(),
                   None if k_norm is None else k_norm.data_ptr(), eps, None if q is None else q_out.data_ptr(), os_)
        return q_out

    def attend(self, batch: KVBatch, q, *, scale: float | None = None, window: int = 0, out=None, ws=None, stream=None):
        """Attention of the batch's rows over their sequences' cached positions (their own included,
        so append first). q (rows, n_heads, head_dim) f32 or of the cache's type; returns out of q's
        shape and type (written there if given; may be q). scale: head_dim ** -0.5 unless given."""
        _require(batch.index == self._index, "the batch and the cache must be on one device")
        qs = self._rows(q, "q", batch.rows, None)
        heads = q.shape[1]
        if out is None:
            with torch.cuda.stream(stream):              # memory that is free on the stream that writes it
                out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        os_ = self._rows(out, "out", batch.rows, heads)
        _require(out.dtype == q.dtype, "out and q must have one type")
        _require(window >= 0, "window must not be negative")
        if ws is None:
            ws = self.workspace(heads, stream)
        _require(ws.get_device() == self._index and ws.is_contiguous(), "the workspace must be dense, on the cache's device")
        self._call(stream, self._attend, batch._ref, _TYPES[q.dtype], heads, q.data_ptr(), qs, out.data_ptr(), os_,
                   self._scale if scale is None else scale, min(window, _ALL), ws.data_ptr(), ws.numel() * ws.element_size())
        return out

    def check(self, stream=None) -> None:
        """Synchronise; raises if a call since the last check met a page id outside the pool, or rows
        or positions outside the batch or its table."""
        self._call(stream, lib().cpg_kv_check)

    def close(self) -> None:
        if self.handle is not None and self.handle.value:
            lib().cpg_kv_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
