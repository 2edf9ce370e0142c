"""The paged cache's ops from their definitions (runtime/paged.py), in numpy and 64 bits: what the
device ops are compared with.  Stored rows are kept as (values, scale) by (page, head, K or V, slot), apart
from any byte layout; ``pack`` turns them into a cache's bytes."""

from __future__ import annotations

import numpy as np

from runtime.paged import CacheLayout

NUMPY = {"float32": np.float32, "float16": np.float16, "int8": np.int8, "float8": np.uint8}


def e4m3_table() -> np.ndarray:
    """The 127 values of e4m3 from zero up, by code."""
    v = [m / 8 * 2.0**-6 for m in range(8)]
    v += [(1 + m / 8) * 2.0**(e - 7) for e in range(1, 16) for m in range(8)]
    return np.array(v[:127])


def row_scale(row: np.ndarray, cache_type: str) -> float:
    amax = float(np.abs(row.astype(np.float64)).max()) if row.size else 0.0
    if not np.isfinite(row).all():
        return float("nan")
    if cache_type in ("int8", "float8"):
        return max(float(np.float32(np.float32(amax) / np.float32(127 if cache_type == "int8" else 448))), 2.0**-126)
    if amax == 0.0:
        return 2.0**-126
    return 2.0**max(int(np.frexp(amax)[1]) - 1 - 14, -126)


def store(row: np.ndarray, cache_type: str) -> tuple[np.ndarray, float]:
    """(stored values, scale) of one row, in 64 bits."""
    s = row_scale(row, cache_type)
    if np.isnan(s):
        return np.zeros(row.shape), s
    y = row.astype(np.float64) / s
    if cache_type == "float16":
        return y.astype(np.float16).astype(np.float64), s
    if cache_type == "int8":
        return np.rint(y), s
    if cache_type == "float8":
        t = e4m3_table()
        a = np.abs(y)
        hi = np.clip(np.searchsorted(t, a), 0, 126)
        lo = np.maximum(hi - 1, 0)
        far = (t[hi] - a) - (a - t[lo])
        at = np.where((far < 0) | ((far == 0) & (hi % 2 == 0)), hi, lo)
        return np.copysign(t[at], y), s
    return y.astype(np.float32).astype(np.float64), s


class Pages:
    """A cache's rows as stored, (values, scale) of [page, head, K or V, slot]; zeros at first."""

    def __init__(self, layout: CacheLayout, n: int) -> None:
        self.layout, self.n = layout, n
        shape = (n, layout.kv_heads, 2, layout.page_size)
        self.y, self.s = np.zeros((*shape, layout.head_dim)), np.zeros(shape, np.float32)

    @classmethod
    def random(cls, layout: CacheLayout, n: int, r: np.random.Generator) -> "Pages":
        """Every row of every page holds something."""
        p = cls(layout, n)
        x = r.standard_normal(p.y.shape) * np.exp(0.5 * r.standard_normal((*p.s.shape, 1)))
        for at in np.ndindex(p.s.shape):
            p.y[at], p.s[at] = store(x[at].astype(np.float32), layout.cache_type)
        return p

    def place(self, table: np.ndarray, b: int, pos: int) -> tuple[int, int] | None:
        size = self.layout.page_size
        if pos < 0 or pos >= table.shape[1] * size:
            return None
        page = int(table[b, pos // size])
        return (page, pos % size) if 0 <= page < self.n else None

    def write(self, k, v, table, start, count) -> None:
        for b in range(k.shape[0]):
            for i in range(min(max(int(count[b]), 0), k.shape[2])):
                at = self.place(table, b, int(start[b]) + i)
                if at is None:
                    continue
                for h in range(k.shape[1]):
                    for j, x in enumerate((k, v)):
                        self.y[at[0], h, j, at[1]], self.s[at[0], h, j, at[1]] = store(x[b, h, i], self.layout.cache_type)

    def rows(self, table, b: int, h: int, j: int, positions) -> np.ndarray:
        """What positions of a sequence stand for, NaN where there is none."""
        out = np.full((len(positions), self.layout.head_dim), np.nan)
        for i, pos in enumerate(positions):
            at = self.place(table, b, int(pos))
            if at is not None:
                out[i] = self.y[at[0], h, j, at[1]] * float(self.s[at[0], h, j, at[1]])
        return out

    def read(self, table, start, count, length: int) -> np.ndarray:
        lay = self.layout
        out = np.zeros((2, table.shape[0], lay.kv_heads, length, lay.head_dim))
        for j in range(2):
            for b in range(table.shape[0]):
                n = min(max(int(count[b]), 0), length)
                for h in range(lay.kv_heads):
                    out[j, b, h, :n] = self.rows(table, b, h, j, range(int(start[b]), int(start[b]) + n))
        return out

    def attention(self, q, table, start, count, scale: float | None = None) -> tuple[np.ndarray, np.ndarray]:
        """(outputs, how far float32 kernels may be off) for Q [B, H, S, head_dim].

        A score is a sum of head_dim products.  With q and the rows split into two 11-bit halves each
        product is off by at most 3·2^-22 of itself (two roundings to 22 bits, one product of low
        halves left out), and a sum in 32 bits by head_dim·2^-24 of the sum of magnitudes: together
        a score is off by d = (3·2^-22 + head_dim·2^-24)·Σ|q k| times the scale, plus 2^-22 of its own
        size in the exponential's argument and 2^-22 relative in its result.  Weights change by a
        factor of at most e^(2d'), which moves an output by at most 2d'·max|v|; the weighted sum itself
        adds 3·2^-22 + n·2^-24 of max|v| for n keys."""
        lay = self.layout
        B, H, S, hd = q.shape
        scale = 1 / np.sqrt(hd) if scale is None else scale
        out, off = np.zeros(q.shape), np.zeros(q.shape)
        for b in range(B):
            n = min(max(int(count[b]), 0), S)
            total = int(start[b]) + n
            for h in range(H):
                if n == 0:
                    continue
                if int(start[b]) < 0:
                    out[b, h, :n] = np.nan
                    continue
                g = h // (H // lay.kv_heads)
                k, v = (self.rows(table, b, g, j, range(total)) for j in range(2))
                for i in range(n):
                    keys = int(start[b]) + i + 1
                    x = q[b, h, i].astype(np.float64) * scale
                    sc = k[:keys] @ x
                    if np.isnan(sc).any() or np.isnan(v[:keys]).any():
                        out[b, h, i] = np.nan
                        continue
                    w = np.exp(sc - sc.max())
                    out[b, h, i] = w @ v[:keys] / w.sum()
                    d = (3 * 2.0**-22 + hd * 2.0**-24) * (np.abs(k[:keys]) @ np.abs(x)).max()
                    d += 2.0**-22 * (np.abs(sc).max() + 2)
                    off[b, h, i] = (2 * d + 3 * 2.0**-22 + keys * 2.0**-24) * np.abs(v[:keys]).max()
        return out, off

    def pack(self) -> np.ndarray:
        """The cache's bytes."""
        lay = self.layout
        kind = NUMPY[lay.cache_type]
        y = np.zeros((*self.y.shape[:-1], lay.row))
        y[..., :lay.head_dim] = self.y
        if lay.cache_type == "float8":
            code = np.searchsorted(e4m3_table(), np.abs(y)).astype(np.uint8)
            y = code | np.where(np.signbit(y), 128, 0).astype(np.uint8)
        y = y.astype(kind)
        out = np.zeros((self.n, lay.kv_heads, lay.head_bytes), np.uint8)
        part = lay.page_size * lay.row * np.dtype(kind).itemsize
        out[..., :part] = np.ascontiguousarray(y[:, :, 0]).reshape(self.n, lay.kv_heads, -1).view(np.uint8)
        v = y[:, :, 1].reshape(self.n, lay.kv_heads, lay.page_size // 8, 8, lay.row).swapaxes(-1, -2)
        out[..., part:2 * part] = np.ascontiguousarray(v).reshape(self.n, lay.kv_heads, -1).view(np.uint8)
        out[..., 2 * part:] = np.ascontiguousarray(self.s).reshape(self.n, lay.kv_heads, -1).view(np.uint8)
        return out.reshape(lay.shape(self.n))


def verify(target, draft, tokens, uniforms, count) -> np.ndarray:
    B, D = tokens.shape
    out = np.full((B, D + 1), -1, np.int64)
    for b in range(B):
        c = min(max(int(count[b]), 0), D)
        n = 0
        while n < c:
            t = int(tokens[b, n])
            if not 0 <= t < target.shape[2]:
                break
            if not float(uniforms[b, n]) * float(draft[b, n, t]) < float(target[b, n, t]):
                break
            out[b, n] = t
            n += 1
        p = target[b, n].astype(np.float64)
        positive = lambda x: np.where(x > 0, x, 0.0)   # noqa: E731
        r = positive(p - draft[b, n].astype(np.float64)) if n < c else positive(p)
        if not r.any():
            r = positive(p)
        if not r.any():
            continue
        run = np.cumsum(r)
        passed = np.flatnonzero((run > float(uniforms[b, D]) * run[-1]) & (r > 0))
        out[b, n] = passed[0] if len(passed) else np.flatnonzero(r > 0)[-1]
    return out
