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
from ._lib import PagedKv

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


def _addr(t):
    return None if t is None else t.data_ptr()


def _check_table(what, cache, table, pos):
    """Returns the batch size and the table's width and row stride."""
    if pos.dim() != 1 or pos.dtype != torch.int64 or pos.device != cache.device or not pos.is_contiguous():
        raise ValueError(f"{what}: pos must be int64 [B] on the cache's device")
    B = pos.shape[0]
    shape, stride = table.shape, table.stride()
    if len(shape) != 2 or shape[0] != B or shape[1] < 1 or (shape[1] > 1 and stride[1] != 1) or \
            table.dtype != torch.int32 or table.device != cache.device:
        raise ValueError(f"{what}: table must be int32 [B, width] on the cache's device")
    return B, shape[1], stride[0]


def _rows(what, t, shape, dtype, device):
    """Returns the address and the token and head strides of rows [T, heads, HD]."""
    stride = t.stride()
    if t.shape != shape or t.dtype != dtype or t.device != device or stride[2] != 1:
        raise ValueError(f"append: {what} must be {dtype} {list(shape)} rows on the cache's device")
    return t.data_ptr(), stride[0], stride[1]


def _vector(what, t, n, dtypes, device):
    if t is None:
        return None
    if t.dtype not in dtypes or t.shape != (n,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"append: {what} must be {dtypes[0]} [{n}] on the cache's device")
    return t.data_ptr()


_NORM = (torch.bfloat16, torch.int16, torch.uint16)
_F32 = (torch.float32,)
_I32 = (torch.int32,)


def append(cache, table, pos, k, v, cu=None, q=None, q_out=None, qn=None, kn=None, inv=None, eps=1e-6):
    """Write the k and v rows [T, KV, HD] (fp32 or bf16, any strides along tokens and heads) of T new tokens to their
    pages. cu (int32 [B+1]): sequence b's tokens are rows cu[b] .. cu[b+1]-1, the first at position pos[b]; rows from
    cu[B] on are left alone. Without cu there is one token per sequence (T == B). qn / kn: q / k norm weights (bf16
    [HD]); inv: fp32 [HD/2] rotation frequencies (None: no rotation, for keys that are rotated already). q [T, H, HD]
    is normed and rotated into q_out (q_out may be q itself). No two tokens may share a cache row."""
    B, width, ld = _check_table("append", cache, table, pos)
    dt = k.dtype
    if dt not in _DT or k.dim() != 3:
        raise ValueError("append: rows must be fp32 or bf16 [T, heads, HD]")
    T, KV, HD, dev = k.shape[0], cache.KV, cache.HD, cache.device
    if (q is None) != (q_out is None):
        raise ValueError("append: q and q_out go together")
    kr, vr = _rows("k", k, (T, KV, HD), dt, dev), _rows("v", v, (T, KV, HD), dt, dev)
    H, qr, qo = 0, (None, 0, 0), (None, 0, 0)
    if q is not None and q.dim() == 3 and q.shape[1]:
        H = q.shape[1]
        qr, qo = _rows("q", q, (T, H, HD), dt, dev), _rows("q_out", q_out, (T, H, HD), dt, dev)
    cu_at = _vector("cu", cu, B + 1, _I32, dev)
    if cu is None and T != B:
        raise ValueError("append: without cu there must be one token per sequence")
    qn_at, kn_at = _vector("qn", qn, HD, _NORM, dev), _vector("kn", kn, HD, _NORM, dev)
    inv_at = _vector("inv", inv, HD // 2, _F32, dev)
    if T == 0 or B == 0:
        return q_out
    with _lib.on_device(dev.index) as stream:
        _lib.call("aib_paged_append", cache.ref, table.data_ptr(), ld, width, pos.data_ptr(), cu_at, B, T, H, *qr, *kr,
                  *vr, *qo, _DT[dt], qn_at, kn_at, inv_at, eps, stream)
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
    B, width, ld = _check_table("attention", cache, table, pos)
    HD, dev, dt = cache.HD, cache.device, q.dtype
    shape = q.shape
    if len(shape) != 3 or shape[0] != B or shape[2] != HD or dt not in _DT or q.device != dev:
        raise ValueError("attention: q must be fp32 or bf16 [B, H, HD] on the cache's device")
    H = shape[1]
    if H % cache.KV:
        raise ValueError("attention: the query heads must be a multiple of the key heads")
    if out is None:
        out = torch.empty(shape, dtype=dt, device=dev)
    elif out.shape != shape or out.dtype != dt or out.device != dev:
        raise ValueError("attention: out must have the shape, type and device of q")
    q_st, out_st = q.stride(), out.stride()
    if q_st[2] != 1 or out_st[2] != 1 or (H > 1 and (q_st[1] != HD or out_st[1] != HD)):
        raise ValueError("attention: the heads of a row must be contiguous")
    if B > 1 and out_st[0] < H * HD:
        raise ValueError("attention: the rows of out must be apart")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (B, H) or lse.device != dev or
                            not lse.is_contiguous()):
        raise ValueError("attention: lse must be fp32 [B, H] on the cache's device")
    if window < 0:
        raise ValueError("attention: window must not be negative")
    if B == 0 or H == 0:
        return out
    if ws is None:
        ws = workspace(B, H, cache)
    elif ws.dtype != torch.uint8 or ws.device != dev or not ws.is_contiguous():
        raise ValueError("attention: ws must come from paged.workspace on the cache's device")
    with _lib.on_device(dev.index) as stream:
        _lib.call("aib_paged_attn", cache.ref, table.data_ptr(), ld, width, pos.data_ptr(), B, H, q.data_ptr(), q_st[0],
                  out.data_ptr(), out_st[0], _DT[dt], _addr(lse), window, HD ** -0.5 if scale is None else scale,
                  ws.data_ptr(), ws.numel(), stream)
    return out
