"""The paged-cache ops as torch ops (namespace ``lbr``), for models that are to be exported.

    torch.ops.lbr.cache_write(cache, k, v, page_table, start, count, page_size, cache_type)
    torch.ops.lbr.cache_read(cache, page_table, start, count, length, kv_heads, head_dim, page_size, cache_type)
    torch.ops.lbr.paged_attention(q, cache, page_table, start, count, kv_heads, page_size, cache_type, scale)
    torch.ops.lbr.verify_draft(target, draft, tokens, uniforms, count)

``cache`` is a uint8 buffer of the model (``register_buffer``) of ``CacheLayout.shape(pages)``, which
``cache_write`` changes in place; the exporter makes it a state of the graph.  What the ops do, and the cache's
bytes, is said in runtime/paged.py.  A cache is not read ahead of a write in one forward: nothing in a graph
would order the two (the graph's validation says so).  Called outside an exported graph they run here, in plain torch and 64 bits, on any
device: for a model's reference, not for speed.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor

from ...paged import CacheLayout, check_op

_KIND = {"float32": torch.float32, "float16": torch.float16, "int8": torch.int8, "float8": torch.float8_e4m3fn}
_RAW = {4: torch.int32, 2: torch.int16, 1: torch.uint8}
_LEAST = 2.0**-126


def _check(op: str, tensors: tuple, attrs: dict) -> None:
    """The ops' own checks; values may be of any floating type here (a model's reference runs in 64 bits)."""
    names = ["float32" if t.is_floating_point() else str(t.dtype).replace("torch.", "") for t in tensors]
    check_op(op, [tuple(t.shape) for t in tensors], names, attrs)


def _views(cache: Tensor, lay: CacheLayout) -> tuple[Tensor, Tensor, Tensor]:
    """The cache's K rows [page, head, slot, column], V groups [page, head, group, column, 8] and scales
    [page, head, K or V, slot], elements as raw integers."""
    n, kind = cache.shape[0], _KIND[lay.cache_type]
    size = torch.empty(0, dtype=kind).element_size()
    part = lay.page_size * lay.row * size
    c = cache.view(n, lay.kv_heads, lay.head_bytes)
    k = c[..., :part].view(_RAW[size]).unflatten(-1, (lay.page_size, lay.row))
    v = c[..., part:2 * part].view(_RAW[size]).unflatten(-1, (lay.page_size // 8, lay.row, 8))
    return k, v, c[..., 2 * part:].view(torch.float32).unflatten(-1, (2, lay.page_size))


def _power(e: Tensor) -> Tensor:
    """2**e of whole numbers, in 64 bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _stored(x: Tensor, cache_type: str) -> tuple[Tensor, Tensor]:
    """Rows [.., head_dim] as the cache's type, and their float32 scales."""
    x = x.float().double()
    top = x.abs().amax(-1)
    fine = torch.isfinite(x).all(-1)
    x, top = torch.where(fine[..., None], x, 0.0), torch.where(fine, top, 0.0)
    if cache_type in ("int8", "float8"):
        # the quotient of two float32 values, rounded to float32 once
        s = (top / (127 if cache_type == "int8" else 448)).float().double().clamp(min=_LEAST)
        y = x / s[..., None]
        if cache_type == "int8":
            y = torch.round(y)
        else:
            step = _power((torch.frexp(y)[1] - 4).clamp(min=-9))
            y = (torch.round(y / step) * step).clamp(-448, 448)
    else:
        s = _power(torch.where(top > 0, torch.frexp(top)[1] - 15, -126).clamp(min=-126))
        y = x / s[..., None]
    return y.float().to(_KIND[cache_type]), torch.where(fine, s, math.nan).float()


def _places(cache: Tensor, table: Tensor, pos: Tensor, lay: CacheLayout) -> tuple[Tensor, Tensor, Tensor]:
    """(there is one, page, slot) of positions [batch, n]."""
    wide = table.shape[1]
    inside = (pos >= 0) & (pos < wide * lay.page_size)
    at = pos.clamp(0, wide * lay.page_size - 1)
    page = table.long().gather(1, at // lay.page_size)
    inside &= (page >= 0) & (page < cache.shape[0])
    return inside, page.clamp(0, cache.shape[0] - 1), at % lay.page_size


def _rows(cache: Tensor, table: Tensor, pos: Tensor, lay: CacheLayout) -> Tensor:
    """K and V [2, batch, kv_heads, n, head_dim] of positions [batch, n] in 64 bits, NaN where there is none."""
    k, v, s = _views(cache, lay)
    there, page, slot = _places(cache, table, pos, lay)
    kind = _KIND[lay.cache_type]
    out = torch.stack([k[page, :, slot].view(kind).double(), v[page, :, slot // 8, :, slot % 8].view(kind).double()])
    out = out * torch.stack([s[page, :, 0, slot], s[page, :, 1, slot]]).double()[..., None]
    return torch.where(there[..., None, None], out, math.nan)[..., :lay.head_dim].transpose(2, 3)


@torch.library.custom_op("lbr::cache_write", mutates_args=("cache",))
def cache_write(cache: Tensor, k: Tensor, v: Tensor, page_table: Tensor, start: Tensor, count: Tensor, page_size: int,
                cache_type: str) -> None:
    lay = CacheLayout(k.shape[1], k.shape[3], page_size, cache_type)
    _check("CACHE_WRITE", (cache, k, v, page_table, start, count), lay.attrs)
    i = torch.arange(k.shape[2], device=k.device)
    there, page, slot = _places(cache, page_table, start.long()[:, None] + i, lay)
    b, i = (there & (i < count.long()[:, None])).nonzero(as_tuple=True)
    page, slot = page[b, i], slot[b, i]
    kp, vp, sp = _views(cache, lay)
    pad = (0, lay.row - lay.head_dim)
    for j, x in enumerate((k, v)):
        y, s = _stored(x[b, :, i], cache_type)
        y = torch.nn.functional.pad(y.view(kp.dtype), pad)
        if j == 0:
            kp[page, :, slot] = y
        else:
            vp[page, :, slot // 8, :, slot % 8] = y
        sp[page, :, j, slot] = s


@cache_write.register_fake
def _(cache, k, v, page_table, start, count, page_size, cache_type):
    return None


@torch.library.custom_op("lbr::cache_read", mutates_args=())
def cache_read(cache: Tensor, page_table: Tensor, start: Tensor, count: Tensor, length: int, kv_heads: int, head_dim: int,
               page_size: int, cache_type: str) -> Tensor:
    lay = CacheLayout(kv_heads, head_dim, page_size, cache_type)
    _check("CACHE_READ", (cache, page_table, start, count), {**lay.attrs, "length": length})
    i = torch.arange(length, device=cache.device)
    out = _rows(cache, page_table, start.long()[:, None] + i, lay)
    return torch.where((i < count.long()[:, None])[:, None, :, None], out, 0.0).float()


@cache_read.register_fake
def _(cache, page_table, start, count, length, kv_heads, head_dim, page_size, cache_type):
    return cache.new_empty((2, page_table.shape[0], kv_heads, length, head_dim), dtype=torch.float32)


@torch.library.custom_op("lbr::paged_attention", mutates_args=())
def paged_attention(q: Tensor, cache: Tensor, page_table: Tensor, start: Tensor, count: Tensor, kv_heads: int,
                    page_size: int, cache_type: str, scale: Optional[float] = None) -> Tensor:
    batch, heads, rows, hd = q.shape
    lay = CacheLayout(kv_heads, hd, page_size, cache_type)
    _check("PAGED_ATTENTION", (q, cache, page_table, start, count), {**lay.attrs, "scale": scale})
    n = count.long().clamp(0, rows)
    if not q.numel() or not int(n.max()):
        return torch.zeros_like(q)
    keys = max(1, int((start.long() + n).max()))
    pos = torch.arange(keys, device=q.device)
    k, v = _rows(cache, page_table, pos.expand(batch, keys), lay)
    bad = k.isnan().any(-1) | v.isnan().any(-1)               # [batch, kv_heads, keys]
    k, v = (torch.where(bad[..., None], 0.0, x) for x in (k, v))
    token = torch.arange(rows, device=q.device)
    last = start.long()[:, None] + token                      # [batch, rows]
    seen = pos <= last[..., None]
    each = heads // kv_heads
    x = q.double().unflatten(1, (kv_heads, each)) * (1 / math.sqrt(hd) if scale is None else scale)
    score = x @ k[:, :, None].transpose(-1, -2).contiguous()
    score = torch.where(seen[:, None, None], score, -math.inf)
    w = torch.exp(score - score.amax(-1, keepdim=True))
    out = (w @ v[:, :, None]) / w.sum(-1, keepdim=True)
    reached = (bad[:, :, None] & seen[:, None]).any(-1) | (last < 0)[:, None]   # [batch, kv_heads, rows]
    reached |= (start < 0)[:, None, None]
    out = torch.where(reached[:, :, None, :, None], math.nan, out).flatten(1, 2)
    return torch.where((token < n[:, None])[:, None, :, None], out, 0.0).to(q.dtype)


@paged_attention.register_fake
def _(q, cache, page_table, start, count, kv_heads, page_size, cache_type, scale=None):
    return q.new_empty(q.shape)


@torch.library.custom_op("lbr::verify_draft", mutates_args=())
def verify_draft(target: Tensor, draft: Tensor, tokens: Tensor, uniforms: Tensor, count: Tensor) -> Tensor:
    _check("VERIFY_DRAFT", (target, draft, tokens, uniforms, count), {})
    batch, most = tokens.shape
    vocab = target.shape[2]
    out = torch.full((batch, most + 1), -1, dtype=torch.int64, device=target.device)
    for b in range(batch):
        n, asked = 0, min(max(int(count[b]), 0), most)
        while n < asked:
            t = int(tokens[b, n])
            # a product of two float32 values is exact in 64 bits
            if not 0 <= t < vocab or not float(uniforms[b, n]) * float(draft[b, n, t]) < float(target[b, n, t]):
                break
            out[b, n] = t
            n += 1
        p = target[b, n].double()
        r = p - draft[b, n].double() if n < asked else p
        r = torch.where(r > 0, r, 0.0)
        if not bool(r.any()):
            r = torch.where(p > 0, p, 0.0)
        if bool(r.any()):
            run = r.cumsum(0)
            passed = ((run > float(uniforms[b, most]) * run[-1]) & (r > 0)).nonzero()
            out[b, n] = passed[0, 0] if len(passed) else (r > 0).nonzero()[-1, 0]
    return out


@verify_draft.register_fake
def _(target, draft, tokens, uniforms, count):
    return tokens.new_empty((tokens.shape[0], tokens.shape[1] + 1))
