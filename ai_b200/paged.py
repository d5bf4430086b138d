"""Paged key-value cache: pages of one pool shared by many sequences, so that a sequence costs the pages it fills and
not `maxt` rows (no reference counterpart; its caches are contiguous, core/engine.py:234-235).

  Cache(k, v)                              one layer's pool: bf16 [pages, KV, page, HD] (views of a larger pool are fine)
  append(cache, table, pos, k, v, ...)     new tokens' keys and values into their pages, q / k norm and position
                                           rotation on the way (the batched qk_rope_cache of a contiguous cache)
  attention(q, cache, table, pos, ...)     attention of one new token per sequence
  Pages(pages, B, width, page, device)     hands pages of the pool to the sequences of a batch

`table` is int32 [B, width]: sequence b's row at position p is row p % page of page table[b, p // page]. `pos` is int64
[B] on the device, so that a captured step can be replayed as the sequences grow; a negative position marks an unused
row of the batch. Positions past the table and page ids outside the pool are left out and recorded in the device
status word (`_lib.status`).
"""
import ctypes as C

import torch

from . import _lib
from ._lib import PagedKv, Rows, ptr, stream_ptr

_DT = {torch.float32: 0, torch.bfloat16: 1}


class Cache:
    """Keys and values of one layer: k, v bf16 CUDA tensors [pages, KV, page, HD] of the same strides (page: a power of
    two; HD 64 or 128, contiguous; 16-byte aligned rows). Either order of the heads and rows in memory will do."""

    def __init__(self, k, v):
        for t in (k, v):
            if t.dim() != 4 or t.dtype != torch.bfloat16 or not t.is_cuda:
                raise ValueError("cache: k and v must be bf16 CUDA tensors [pages, KV, page, HD]")
        if k.shape != v.shape or k.stride() != v.stride() or k.device != v.device:
            raise ValueError("cache: k and v must have the same shape, strides and device")
        self.pages, self.KV, self.page, self.HD = k.shape
        if self.HD not in (64, 128) or self.page < 1 or self.page & (self.page - 1) or not self.pages or not self.KV:
            raise ValueError("cache: HD must be 64 or 128 and the rows of a page a power of two")
        if k.stride(3) != 1 or any(s % 8 for s in k.stride()[:3]) or (k.data_ptr() | v.data_ptr()) % 16:
            raise ValueError("cache: rows must be contiguous and 16-byte aligned")
        self.k, self.v, self.device = k, v, k.device
        self.desc = PagedKv(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), self.pages, self.page,
                            self.KV, self.HD)
        self.ref = C.byref(self.desc)


def _check_table(what, cache, table, pos):
    B = pos.shape[0]
    if table.dim() != 2 or table.shape[0] != B or table.dtype != torch.int32 or table.device != cache.device or \
            table.shape[1] < 1 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"{what}: table must be int32 [B, width] on the cache's device")
    if pos.dim() != 1 or pos.dtype != torch.int64 or pos.device != cache.device or (B > 1 and pos.stride(0) != 1):
        raise ValueError(f"{what}: pos must be int64 [B] on the cache's device")
    return B


def _rows(what, t, T, heads, HD, dtype, device):
    if t.dim() != 3 or t.shape[0] != T or t.shape[2] != HD or (heads and t.shape[1] != heads) or t.dtype != dtype or \
            t.device != device or t.stride(2) != 1:
        raise ValueError(f"append: {what} must be [T, heads, HD] rows like k on the cache's device")
    return Rows(t.data_ptr(), t.stride(0), t.stride(1))


def _norm(what, w, HD, device):
    if w is None:
        return None
    if w.dtype not in (torch.bfloat16, torch.int16, torch.uint16) or w.shape != (HD,) or w.device != device or \
            w.stride(0) != 1:
        raise ValueError(f"append: {what} must be bf16 [HD] on the cache's device")
    return ptr(w)


def append(cache, table, pos, k, v, cu=None, q=None, q_out=None, qn=None, kn=None, inv=None, eps=1e-6):
    """Write the k and v rows [T, KV, HD] (fp32 or bf16, any strides along tokens and heads) of T new tokens to their
    pages. cu (int32 [B+1]): sequence b's tokens are rows cu[b] .. cu[b+1]-1, the first at position pos[b]; rows from
    cu[B] on are left alone. Without cu there is one token per sequence (T == B). qn / kn: q / k norm weights (bf16
    [HD]); inv: fp32 [HD/2] rotation frequencies (None: no rotation, for keys that are rotated already). q [T, H, HD]
    is normed and rotated into q_out (q_out may be q itself). No two tokens may share a cache row."""
    B = _check_table("append", cache, table, pos)
    if k.dtype not in _DT:
        raise ValueError("append: rows must be fp32 or bf16")
    T, HD, dev, dt = k.shape[0], cache.HD, cache.device, k.dtype
    if T == 0 or B == 0:
        return q_out
    kr, vr = _rows("k", k, T, cache.KV, HD, dt, dev), _rows("v", v, T, cache.KV, HD, dt, dev)
    if (q is None) != (q_out is None):
        raise ValueError("append: q and q_out go together")
    H, qr, qo = 0, None, None
    if q is not None:
        qr, qo = _rows("q", q, T, 0, HD, dt, dev), _rows("q_out", q_out, T, q.shape[1], HD, dt, dev)
        H = q.shape[1]
        qr, qo = (C.byref(qr), C.byref(qo)) if H else (None, None)
    if cu is None:
        if T != B:
            raise ValueError("append: without cu there must be one token per sequence")
    elif cu.dtype != torch.int32 or cu.shape != (B + 1,) or cu.device != dev or cu.stride(0) != 1:
        raise ValueError("append: cu must be int32 [B + 1] on the cache's device")
    if inv is not None and (inv.dtype != torch.float32 or inv.shape != (HD // 2,) or inv.device != dev or
                            inv.stride(0) != 1):
        raise ValueError("append: inv must be fp32 [HD/2] on the cache's device")
    with _lib.device_of(k):
        _lib.call("aib_paged_append", cache.ref, ptr(table), table.stride(0), table.shape[1], ptr(pos), ptr(cu), B, T, H,
                  qr, C.byref(kr), C.byref(vr), qo, _DT[dt], _norm("qn", qn, HD, dev), _norm("kn", kn, HD, dev),
                  ptr(inv), eps, stream_ptr())
    return q_out


def workspace(B, H, cache):
    """Scratch of `attention` for up to B sequences and H query heads (zero-filled once; calls leave it reusable). Calls
    that may overlap on the GPU need separate ones."""
    n = _lib.lib().aib_paged_attn_workspace(B, H, cache.KV, cache.HD)
    return torch.zeros(max(n, 16), dtype=torch.uint8, device=cache.device)


def attention(q, cache, table, pos, out=None, scale=None, window=0, lse=None, ws=None):
    """Attention of one new token per sequence: q [B, H, HD] (fp32 or bf16, heads contiguous; normed and rotated), its
    own key and value already in the cache at pos[b]. Attends positions 0 .. pos[b], or with a window the last `window`
    of them. out: [B, H, HD] like q (allocated when None); lse: optional fp32 [B, H], the log of the summed
    exponentials; scale: default HD ** -0.5; ws: from `workspace` (a fresh one per call when None). A row that attends
    nothing gives zeros and lse -inf. Returns out."""
    B = _check_table("attention", cache, table, pos)
    HD, dev = cache.HD, cache.device
    if q.dim() != 3 or q.shape[0] != B or q.shape[2] != HD or q.dtype not in _DT or q.device != dev:
        raise ValueError("attention: q must be fp32 or bf16 [B, H, HD] on the cache's device")
    H = q.shape[1]
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if B == 0 or H == 0:
        return out
    if H % cache.KV:
        raise ValueError("attention: the query heads must be a multiple of the key heads")
    if out.shape != q.shape or out.dtype != q.dtype or out.device != dev:
        raise ValueError("attention: out must have the shape, type and device of q")
    for t in (q, out):
        if t.stride(2) != 1 or (H > 1 and t.stride(1) != HD):
            raise ValueError("attention: the heads of a row must be contiguous")
    if B > 1 and out.stride(0) < H * HD:
        raise ValueError("attention: the rows of out must be apart")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (B, H) or lse.device != dev or
                            not lse.is_contiguous()):
        raise ValueError("attention: lse must be fp32 [B, H] on the cache's device")
    if window < 0:
        raise ValueError("attention: window must not be negative")
    with _lib.device_of(q):
        if ws is None:
            ws = workspace(B, H, cache)
        _lib.call("aib_paged_attn", cache.ref, ptr(table), table.stride(0), table.shape[1], ptr(pos), B, H, ptr(q),
                  q.stride(0), ptr(out), out.stride(0), _DT[q.dtype], ptr(lse), window,
                  HD ** -0.5 if scale is None else scale, ptr(ws), ws.numel(), stream_ptr())
    return out
