"""A paged cache of keys and values held in 4 bits, and attention over it.

The cache is one uint8 tensor ``data`` [pages, kv_heads, page / 16, tile], a
tile being 16 tokens of one head: key codes [d / group][16][group / 2], value
codes [d / 2][16] (token t in column 4 ((t & 7) >> 1) + 2 (t & 1) + (t >> 3)),
then float16 (scale, zero) pairs [d / group][16] of the keys and of the values;
a code c stands for c * scale + zero (include/st_b200.h, st_kv4_append).  Slot s
is token s % page of page s // page.  ``empty`` makes one; ``append`` writes
new tokens into it (rotating keys and queries by position on the way),
``read`` takes tokens out again and ``attend`` is attention over it: single
tokens, a few guessed ahead, or pieces of prompts.

Calls run on torch's current stream.  What only the device knows (a length, a
slot or a page number out of range) is reported by ``handle().sync()``.  There
is no counterpart in the reference, whose sequences always run whole.
"""
import ctypes

import torch

from . import _native as N
from .device import handle, ptr

_DTYPES = {torch.float32: N.ST_F32, torch.float16: N.ST_F16, torch.bfloat16: N.ST_BF16}


def tile_bytes(d: int, group: int) -> int:
    """Bytes of a tile: 16 tokens of one head."""
    return 16 * d + 128 * (d // group)


def empty(pages: int, page: int, kv_heads: int, d: int, group: int = 64, device=None) -> torch.Tensor:
    """A cache of ``pages`` pages of ``page`` tokens (a multiple of 16)."""
    if page % 16:
        raise ValueError("a page of %d tokens does not split into tiles of 16" % page)
    dev = torch.device("cuda") if device is None else device
    return torch.zeros((pages, kv_heads, page // 16, tile_bytes(d, group)), dtype=torch.uint8, device=dev)


def _cache(data: torch.Tensor, d: int, group: int):
    if data.dtype != torch.uint8 or data.dim() != 4 or not data.is_contiguous() or not data.is_cuda:
        raise ValueError("the cache is a contiguous uint8 CUDA tensor [pages, kv_heads, page / 16, tile]")
    if group < 1 or d % group or data.shape[3] != tile_bytes(d, group):
        raise ValueError("tiles of %d bytes do not hold heads of %d in groups of %d" % (data.shape[3], d, group))
    return data.shape[0], data.shape[2] * 16, data.shape[1]


def _whole(t: torch.Tensor, dtype, like: torch.Tensor, name: str, shape=None):
    if t.dtype != dtype or not t.is_contiguous() or t.device != like.device:
        raise ValueError("%s must be a contiguous %s tensor on %s" % (name, str(dtype)[6:], like.device))
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError("%s has shape %s, not %s" % (name, tuple(t.shape), tuple(shape)))
    return t


def _rows(t: torch.Tensor, dtype, like: torch.Tensor, name: str, shape):
    """t [n, heads, d] with contiguous rows of d (any strides between them)."""
    if t.dtype != dtype or t.device != like.device:
        raise ValueError("%s must be a %s tensor on %s" % (name, str(dtype)[6:], like.device))
    if tuple(t.shape) != tuple(shape):
        raise ValueError("%s has shape %s, not %s" % (name, tuple(t.shape), tuple(shape)))
    return t if t.stride(2) == 1 else t.contiguous()


def append(data: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, group: int = 64, q=None,
           cos=None, sin=None, positions=None, interleaved: bool = False, out=None):
    """Writes tokens k, v [n, kv_heads, d] (float32, float16 or bfloat16) to ``slots`` (int64 [n], all different;
    negative: left out).  With cos and sin (float32 [positions, rotary / 2]) and ``positions`` (int32 [n]) the first
    ``rotary`` channels of the keys are rotated first, and those of q [n, heads, d], which is returned (into ``out``)."""
    n, kv_heads, d = k.shape
    pages, page, have = _cache(data, d, group)
    dtype = k.dtype
    if dtype not in _DTYPES:
        raise ValueError("keys in %s" % dtype)
    k = _rows(k, dtype, data, "k", (n, have, d))
    v = _rows(v, dtype, data, "v", (n, have, d))
    _whole(slots, torch.int64, data, "slots", (n,))
    rotary, table, heads, qs = 0, 0, 0, (0, 0)
    if cos is not None:
        table, rotary = cos.shape[0], 2 * cos.shape[1]
        _whole(cos, torch.float32, data, "cos"), _whole(sin, torch.float32, data, "sin", cos.shape)
        _whole(positions, torch.int32, data, "positions", (n,))
    if q is not None:
        if cos is None:
            raise ValueError("queries are only rotated: without cos and sin there is nothing to do")
        heads = q.shape[1]
        q = _rows(q, dtype, data, "q", (n, heads, d))
        qs = q.stride()
        out = torch.empty((n, heads, d), dtype=dtype, device=q.device) if out is None else \
            _whole(out, dtype, data, "out", (n, heads, d))
    handle(data.device).call("st_kv4_append", ptr(data), pages, page, kv_heads, d, group, ptr(k), k.stride(0),
                             k.stride(1), ptr(v), v.stride(0), v.stride(1), ptr(slots), n, ptr(q), qs[0], qs[1],
                             ptr(out) if q is not None else None, heads, ptr(cos), ptr(sin),
                             ptr(positions) if rotary else None, table, rotary, int(interleaved), _DTYPES[dtype])
    return out if q is not None else None


def read(data: torch.Tensor, slots: torch.Tensor, d: int, group: int = 64, dtype=torch.float32, out=None):
    """-> (k, v) [n, kv_heads, d]: what the cache holds in ``slots`` (int64 [n]; negative: zeros)."""
    pages, page, kv_heads = _cache(data, d, group)
    if dtype not in _DTYPES:
        raise ValueError("values in %s" % dtype)
    _whole(slots, torch.int64, data, "slots", slots.shape[:1])
    shape = (slots.shape[0], kv_heads, d)
    if out is None:
        out = (torch.empty(shape, dtype=dtype, device=data.device), torch.empty(shape, dtype=dtype,
                                                                                device=data.device))
    _whole(out[0], dtype, data, "out[0]", shape), _whole(out[1], dtype, data, "out[1]", shape)
    handle(data.device).call("st_kv4_read", ptr(data), pages, page, kv_heads, d, group, ptr(slots), shape[0],
                             ptr(out[0]), ptr(out[1]), _DTYPES[dtype])
    return out


def attend(q: torch.Tensor, data: torch.Tensor, pages: torch.Tensor, kv_len: torch.Tensor, scale: float,
           group: int = 64, q_start=None, max_q=None, causal: bool = True, one: bool = False, window: int = 0,
           return_lse: bool = False, out=None):
    """-> o [rows, heads, d] of q's type, with ``return_lse`` also lse float32 [rows, heads].

    q [rows, heads, d]: sequence b has rows q_start[b] .. q_start[b + 1] (int32 [batch + 1]; None: one row for each
    sequence), at most ``max_q`` (None: the number of rows), its last ones by position; its kv_len[b] (int32) keys
    lie in pages[b] (int32 [batch, most]).  ``causal``: a row sees the keys up to its own position; ``window``: only
    the last ``window`` of them; ``one``: softmax1.  A row that sees nothing gives 0 (lse -inf; softmax1: 0)."""
    rows, heads, d = q.shape
    n_pages, page, kv_heads = _cache(data, d, group)
    dtype = q.dtype
    if dtype not in _DTYPES:
        raise ValueError("queries in %s" % dtype)
    if heads % kv_heads:
        raise ValueError("%d heads do not share %d" % (heads, kv_heads))
    q = _rows(q, dtype, data, "q", (rows, heads, d))
    batch = kv_len.shape[0]
    _whole(kv_len, torch.int32, data, "kv_len", (batch,))
    _whole(pages, torch.int32, data, "pages", (batch, pages.shape[-1]))
    if q_start is not None:
        _whole(q_start, torch.int32, data, "q_start", (batch + 1,))
        max_q = rows if max_q is None else max_q
    elif rows != batch:
        raise ValueError("%d rows for %d sequences: q_start says whose they are" % (rows, batch))
    else:
        max_q = 1
    if window < 0 or (rows and max_q < 1):
        raise ValueError("window %d, max_q %d" % (window, max_q))
    o = torch.empty((rows, heads, d), dtype=dtype, device=q.device) if out is None else \
        _whole(out, dtype, data, "out", (rows, heads, d))
    lse = torch.empty((rows, heads), dtype=torch.float32, device=q.device) if return_lse else None
    if rows and batch:
        h = handle(data.device)
        need = ctypes.c_int64()
        h.call("st_kv4_attn_workspace", batch, rows, max_q, pages.shape[1] * page, heads, kv_heads, d, ctypes.byref(need))
        # torch's allocator gives each stream, and each captured graph, a workspace of its own
        work = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
        h.call("st_kv4_attn", ptr(q), q.stride(0), q.stride(1), ptr(o), ptr(lse), ptr(data), n_pages, page, heads,
               kv_heads, d, group, ptr(pages), pages.shape[1], ptr(kv_len), ptr(q_start), batch, rows, max_q,
               float(scale), int(causal), int(one), window, _DTYPES[dtype], ptr(work), need.value)
    return (o, lse) if return_lse else o
