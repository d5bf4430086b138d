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
        within = self.HD  # from the smallest stride on, every one steps over all that lies within it
        for s, n in sorted(zip(k.stride()[:3], k.shape[:3])):
            if n > 1 and s < within:
                raise ValueError("cache: rows must not overlap")
            within += (n - 1) * s
        self.k, self.v, self.device, self.index = k, v, k.device, k.get_device()
        self.desc = PagedKv(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), self.pages, self.page,
                            self.KV, self.HD)
        self.ref = C.byref(self.desc)


class Pages:
    """The pages of a pool and the table of a batch: `table` int32 [B, width] on the device, a sequence's pages in the
    order of its rows (entries that it does not have are -1)."""

    def __init__(self, pages, B, width, page, device):
        if pages < 1 or B < 1 or width < 1 or page < 1:
            raise ValueError("pages, sequences, width and rows per page must be positive")
        self.total, self.page, self.width = pages, page, width
        self.left = list(range(pages - 1, -1, -1))
        self.held = [[] for _ in range(B)]
        self.table = torch.full((B, width), -1, dtype=torch.int32, device=device)

    def grow(self, b, rows):
        """Give sequence b the pages that `rows` rows need, all of them or none."""
        need = -(-rows // self.page) - len(self.held[b])
        if need <= 0:
            return
        if len(self.held[b]) + need > self.width:
            raise ValueError(f"{rows} rows do not fit a table of {self.width} pages")
        if need > len(self.left):
            raise ValueError(f"{need} pages are needed, {len(self.left)} are free")
        new = [self.left.pop() for _ in range(need)]
        at = len(self.held[b])
        self.held[b] += new
        self.table[b, at:at + need] = torch.tensor(new, dtype=torch.int32, device=self.table.device)

    def free(self, b):
        """Take sequence b's pages back."""
        self.left += reversed(self.held[b])
        self.held[b] = []
        self.table[b] = -1


def _addr(t):
    return None if t is None else t.data_ptr()


def _check_table(what, cache, table, pos):
    """Returns the batch size and the table's width and row stride."""
    if pos.dim() != 1 or pos.dtype is not torch.int64 or pos.get_device() != cache.index or not pos.is_contiguous():
        raise ValueError(f"{what}: pos must be int64 [B] on the cache's device")
    B, = pos.shape
    if table.dim() != 2 or table.dtype is not torch.int32 or table.get_device() != cache.index:
        raise ValueError(f"{what}: table must be int32 [B, width] on the cache's device")
    rows, width = table.shape
    ld, step = table.stride()
    if rows != B or width < 1 or (width > 1 and step != 1):
        raise ValueError(f"{what}: table must be int32 [B, width] on the cache's device")
    return B, width, ld


def _rows(what, t, T, heads, cache, dtype):
    """Returns the address and the token and head strides of rows [T, heads, HD]."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[2] != cache.HD or shape[1] != heads or shape[0] != T or stride[2] != 1 or \
            t.dtype is not dtype or t.get_device() != cache.index:
        raise ValueError(f"append: {what} must be {dtype} [{T}, {heads}, {cache.HD}] rows on the cache's device")
    return t.data_ptr(), stride[0], stride[1]


def _vector(what, t, n, dtypes, index):
    """Returns the address of n contiguous elements."""
    if t.dtype not in dtypes or t.numel() != n or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"append: {what} must be {dtypes[0]} [{n}] on the cache's device")
    return t.data_ptr()


_NORM = (torch.bfloat16, torch.int16, torch.uint16)
_F32 = (torch.float32,)
_I32 = (torch.int32,)
_NO_ROWS = (None, 0, 0)
_NO_WINDOW = 2 ** 63 - 1  # of C's type; longer than any cache


def append(cache, table, pos, k, v, cu=None, q=None, q_out=None, qn=None, kn=None, inv=None, eps=1e-6):
    """Write the k and v rows [T, KV, HD] (fp32 or bf16, any strides along tokens and heads) of T new tokens to their
    pages. cu (int32 [B+1]): sequence b's tokens are rows cu[b] .. cu[b+1]-1, the first at position pos[b]; rows from
    cu[B] on are left alone. Without cu there is one token per sequence (T == B). qn / kn: q / k norm weights (bf16
    [HD]); inv: fp32 [HD/2] rotation frequencies (None: no rotation, for keys that are rotated already). q [T, H, HD]
    is normed and rotated into q_out (q itself, or memory that it shares with none of q, k and v). No two tokens may share a cache row."""
    B, width, ld = _check_table("append", cache, table, pos)
    dt = k.dtype
    if dt not in _DT or k.dim() != 3:
        raise ValueError("append: rows must be fp32 or bf16 [T, heads, HD]")
    T, HD = k.shape[0], cache.HD
    if (q is None) != (q_out is None):
        raise ValueError("append: q and q_out go together")
    H, qr, qo = 0, _NO_ROWS, _NO_ROWS
    if q is not None:
        if q.dim() != 3:
            raise ValueError("append: q must be [T, heads, HD] rows like k")
        H = q.shape[1]
    if H:
        qr, qo = _rows("q", q, T, H, cache, dt), _rows("q_out", q_out, T, H, cache, dt)
    kr, vr = _rows("k", k, T, cache.KV, cache, dt), _rows("v", v, T, cache.KV, cache, dt)
    if cu is None and T != B:
        raise ValueError("append: without cu there must be one token per sequence")
    index = cache.index
    cu_at = None if cu is None else _vector("cu", cu, B + 1, _I32, index)
    inv_at = None if inv is None else _vector("inv", inv, HD // 2, _F32, index)
    qn_at = None if qn is None else _vector("qn", qn, HD, _NORM, index)
    kn_at = None if kn is None else _vector("kn", kn, HD, _NORM, index)
    if T == 0 or B == 0:
        return q_out
    with _lib.on_device(index) as stream:
        _lib.call("aib_paged_append", cache.ref, table.data_ptr(), ld, width, pos.data_ptr(), cu_at, B, T, H, *qr, *kr,
                  *vr, *qo, _DT[dt], qn_at, kn_at, inv_at, eps, stream)
    return q_out


def workspace(B, H, cache):
    """Scratch of `attention` for up to B sequences and H query heads (zero-filled once; calls leave it reusable). Calls
    that may overlap on the GPU need separate ones. After a device status of 101 (a wait that ran out) it has to be
    zeroed again."""
    n = _lib.lib().aib_paged_attn_workspace(B, H, cache.KV, cache.HD)
    return torch.zeros(max(n, 16), dtype=torch.uint8, device=cache.device)


def attention(q, cache, table, pos, out=None, scale=None, window=0, lse=None, ws=None):
    """Attention of one new token per sequence (at most 4096): q [B, H, HD] (fp32 or bf16, heads contiguous; normed and
    rotated), its own key and value already in the cache at pos[b]. Attends positions 0 .. pos[b], or with a window the last `window`
    of them. out: [B, H, HD] like q (allocated when None; not q itself); lse: optional fp32 [B, H], the log of the summed
    exponentials; scale: default HD ** -0.5; ws: from `workspace` (a fresh one per call when None). A row that attends
    nothing gives zeros and lse -inf; a head whose scores are all -inf gives NaN and lse -inf. Infinite queries, and
    infinite keys or values in attended rows, may give NaN where they meet. Returns out."""
    B, width, ld = _check_table("attention", cache, table, pos)
    HD, index, dt = cache.HD, cache.index, q.dtype
    if q.dim() != 3 or dt not in _DT or q.get_device() != index:
        raise ValueError("attention: q must be fp32 or bf16 [B, H, HD] on the cache's device")
    n, H, d = q.shape
    if n != B or d != HD:
        raise ValueError("attention: q must be fp32 or bf16 [B, H, HD] on the cache's device")
    if H % cache.KV:
        raise ValueError("attention: the query heads must be a multiple of the key heads")
    if out is None:
        out = torch.empty(q.shape, dtype=dt, device=cache.device)
    elif out.shape != q.shape or out.dtype is not dt or out.get_device() != index:
        raise ValueError("attention: out must have the shape, type and device of q")
    (q_ld, q_hs, q_step), (out_ld, out_hs, out_step) = q.stride(), out.stride()
    if q_step != 1 or out_step != 1 or (H > 1 and (q_hs != HD or out_hs != HD)):
        raise ValueError("attention: the heads of a row must be contiguous")
    if B > 1 and out_ld < H * HD:
        raise ValueError("attention: the rows of out must be apart")
    if lse is not None and (lse.dtype is not torch.float32 or lse.shape != (B, H) or lse.get_device() != index or
                            not lse.is_contiguous()):
        raise ValueError("attention: lse must be fp32 [B, H] on the cache's device")
    if window < 0:
        raise ValueError("attention: window must not be negative")
    if B == 0 or H == 0:
        return out
    if ws is None:
        ws = workspace(B, H, cache)
    elif ws.dtype is not torch.uint8 or ws.get_device() != index or not ws.is_contiguous():
        raise ValueError("attention: ws must come from paged.workspace on the cache's device")
    with _lib.on_device(index) as stream:
        _lib.call("aib_paged_attn", cache.ref, table.data_ptr(), ld, width, pos.data_ptr(), B, H, q.data_ptr(), q_ld,
                  out.data_ptr(), out_ld, _DT[dt], _addr(lse), min(window, _NO_WINDOW), HD ** -0.5 if scale is None else scale,
                  ws.data_ptr(), ws.numel(), stream)
    return out
