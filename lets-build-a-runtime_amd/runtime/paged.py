"""The paged key/value cache: its types, its layout, and what the ops over it take.

A cache is a uint8 state ``[pages, page_bytes]`` (``CacheLayout.shape``), one for each layer.
A page holds ``page_size`` token positions of every K/V head; a sequence's positions lie in the
pages that its row of the page table names, in order.  Inside a page, for each head in turn:

* the K rows, ``[page_size][hdp]`` (``hdp``: ``head_dim`` rounded up to 16, the rest zeros);
* the V rows in groups of eight positions, ``[page_size / 8][hdp][8]``: the eight positions of one
  column side by side are what the matrix cores take for the product with the weights;
* a float32 scale for each K row, then one for each V row.

A stored value stands for itself times its row's scale (a row: one position of one head):

* ``float32``, ``float16``: the scale is the power of two that brings the row's largest magnitude
  into [2^14, 2^15), at least 2^-126.  ``float32`` keeps every value that is not 2^100 times smaller
  than its row's largest; ``float16`` rounds to 11 bits, and neither overflows nor loses bits of
  rows of small values;
* ``int8``: the scale is the largest magnitude / 127, at least 2^-126; values to the nearest whole
  multiple, ties to even;
* ``float8`` (e4m3): the same with 448, and e4m3's values.

A row that holds an infinity or a NaN is stored as zeros with a NaN scale: it reads back as NaN,
and every output that attends to it is NaN.

The ops (graph nodes; every index tensor int32):

* ``CACHE_WRITE [cache, K, V, page_table, start, count]``: rows i < count[b] of K, V
  ``[B, kv_heads, S, head_dim]`` go to positions start[b] + i.  Positions outside the table and
  rows whose page is not one of the cache's are dropped.  Sequences written in one call share no
  page that both write.  The output is the cache itself.
* ``CACHE_READ [cache, page_table, start, count]``, ``length``: float32 ``[2, B, kv_heads, length,
  head_dim]``, K then V of positions start[b] + i for i < count[b], zeros behind them.
* ``PAGED_ATTENTION [Q, cache, page_table, start, count]``: row i < count[b] of Q
  ``[B, heads, S, head_dim]`` attends to positions 0 .. start[b] + i (the chunk's own rows have been
  written before), query head h to K/V head h // (heads // kv_heads); rows i >= count[b] are zeros.
* ``VERIFY_DRAFT [target, draft, tokens, uniforms, count]``: tokens ``[B, D]`` (int64) were drawn
  from draft ``[B, D, V]``; target ``[B, D + 1, V]`` are the model's own probabilities.  Token i <
  count[b] stands while uniforms[b, i] * draft[token] < target[token] and all before it do; behind the
  n that stand comes one drawn with uniforms[b, D]: from max(target - draft, 0) of row n, or from the
  target's row where all count[b] stand or that difference is zero everywhere (the first index whose
  running sum, in 64 bits, passes uniforms[b, D] times the whole).  Output: int64 ``[B, D + 1]``,
  the n tokens, the drawn one, then -1.  A row without a probability above zero gives -1.

counts are taken as 0 .. S (``length``, D).  A table's row reaches 2^30 positions at most.  Positions a
table does not reach, and pages that the cache does not have, read as NaN.
"""

from __future__ import annotations

from dataclasses import dataclass

# cache_type -> (code in OpNode.extra, bytes of an element)
CACHE_TYPES: dict[str, tuple[int, int]] = {"float32": (0, 4), "float16": (1, 2), "int8": (2, 1), "float8": (3, 1)}

MAX_HEAD_DIM = 256
PAGE_SIZES = (16, 32768)    # powers of two from .. to


@dataclass(frozen=True)
class CacheLayout:
    """Sizes of one layer's cache."""
    kv_heads: int
    head_dim: int
    page_size: int
    cache_type: str = "float32"

    def __post_init__(self) -> None:
        if self.cache_type not in CACHE_TYPES:
            raise ValueError(f"cache_type '{self.cache_type}' is none of {', '.join(CACHE_TYPES)}")
        if not 1 <= self.head_dim <= MAX_HEAD_DIM:
            raise ValueError(f"head_dim {self.head_dim} is not in 1 .. {MAX_HEAD_DIM}")
        if self.kv_heads < 1:
            raise ValueError(f"kv_heads {self.kv_heads} is not positive")
        p = self.page_size
        if not PAGE_SIZES[0] <= p <= PAGE_SIZES[1] or p & (p - 1):
            raise ValueError(f"page_size {p} is not a power of two from {PAGE_SIZES[0]} to {PAGE_SIZES[1]}")
        if self.page_bytes >= 2**31:
            raise ValueError(f"a page of {self.page_bytes} bytes is larger than 2 GiB")

    @classmethod
    def of(cls, attrs: dict) -> "CacheLayout":
        """The layout that a cache op's attributes name."""
        missing = [k for k in ("kv_heads", "head_dim", "page_size") if k not in attrs]
        if missing:
            raise ValueError(f"a cache op needs the attribute '{missing[0]}'")
        return cls(attrs["kv_heads"], attrs["head_dim"], attrs["page_size"], attrs.get("cache_type", "float32"))

    @property
    def attrs(self) -> dict:
        """The attributes of a cache op over this layout."""
        return {"kv_heads": self.kv_heads, "head_dim": self.head_dim, "page_size": self.page_size,
                "cache_type": self.cache_type}

    @property
    def row(self) -> int:
        """Stored columns of a row."""
        return (self.head_dim + 15) // 16 * 16

    @property
    def head_bytes(self) -> int:
        return self.page_size * (2 * self.row * CACHE_TYPES[self.cache_type][1] + 8)

    @property
    def page_bytes(self) -> int:
        return self.kv_heads * self.head_bytes

    def shape(self, pages: int) -> tuple[int, int]:
        """Shape of the uint8 state that holds `pages` pages."""
        return (pages, self.page_bytes)


# ---------------------------------------------------------------- what the ops take

# (name, dtype, rank) of each input; the cache's dims are the layout's
_CACHE, _TABLE = ("cache", "uint8", 2), [("page_table", "int32", 2), ("start", "int32", 1), ("count", "int32", 1)]
INPUTS = {
    "CACHE_WRITE": [_CACHE, ("K", "float32", 4), ("V", "float32", 4), *_TABLE],
    "CACHE_READ": [_CACHE, *_TABLE],
    "PAGED_ATTENTION": [("Q", "float32", 4), _CACHE, *_TABLE],
    "VERIFY_DRAFT": [("target", "float32", 3), ("draft", "float32", 3), ("tokens", "int64", 2),
                     ("uniforms", "float32", 2), ("count", "int32", 1)],
}
OUT_DTYPE = {"CACHE_WRITE": "uint8", "CACHE_READ": "float32", "PAGED_ATTENTION": "float32", "VERIFY_DRAFT": "int64"}


def check_op(op: str, shapes: list[tuple], dtypes: list[str], attrs: dict, out_shape: tuple | None = None,
             out_dtype: str | None = None) -> None:
    """Raise ValueError if a node's inputs and attributes do not fit its op."""
    want = INPUTS[op]
    if len(shapes) != len(want):
        raise ValueError(f"{op} takes {len(want)} inputs ({', '.join(n for n, _, _ in want)}), got {len(shapes)}")
    by = {}
    for (name, dtype, rank), shape, have in zip(want, shapes, dtypes):
        if have != dtype:
            raise ValueError(f"{op}: {name} is {have}, expected {dtype}")
        if len(shape) != rank:
            raise ValueError(f"{op}: {name} has shape {tuple(shape)}, expected {rank} dims")
        by[name] = tuple(shape)

    def same(name, shape):
        if by[name] != shape:
            raise ValueError(f"{op}: {name} has shape {by[name]}, expected {shape}")

    if op == "VERIFY_DRAFT":
        batch, d = by["tokens"]
        vocab = by["target"][2]
        if vocab < 1:
            raise ValueError(f"{op}: the vocabulary is empty")
        same("target", (batch, d + 1, vocab))
        same("draft", (batch, d, vocab))
        same("uniforms", (batch, d + 1))
        same("count", (batch,))
        out = (batch, d + 1)
    else:
        lay = CacheLayout.of(attrs)
        if by["cache"][1] != lay.page_bytes:
            raise ValueError(f"{op}: pages of the cache have {by['cache'][1]} bytes, {lay} has {lay.page_bytes}")
        if by["cache"][0] < 1 or by["page_table"][1] < 1:
            raise ValueError(f"{op}: the cache and the page table need a page")
        if by["page_table"][1] * lay.page_size > 2**30:
            raise ValueError(f"{op}: a table of {by['page_table'][1]} pages reaches positions past 2^30")
        batch = by["page_table"][0]
        same("start", (batch,))
        same("count", (batch,))
        if op == "CACHE_WRITE":
            same("K", (batch, lay.kv_heads, by["K"][2], lay.head_dim))
            same("V", by["K"])
            out = by["cache"]
        elif op == "CACHE_READ":
            length = attrs.get("length")
            if not isinstance(length, int) or length < 0:
                raise ValueError(f"{op}: length {length!r} is not a whole number from 0")
            out = (2, batch, lay.kv_heads, length, lay.head_dim)
        else:
            heads = by["Q"][1]
            same("Q", (batch, heads, by["Q"][2], lay.head_dim))
            if heads % lay.kv_heads or not heads:
                raise ValueError(f"{op}: {heads} query heads over {lay.kv_heads} K/V heads")
            scale = attrs.get("scale")
            if scale is not None and not 0.0 < scale < float("inf"):
                raise ValueError(f"{op}: scale {scale!r} is not a positive number")
            out = by["Q"]
    if out_shape is not None and tuple(out_shape) != out:
        raise ValueError(f"{op}: the output has shape {tuple(out_shape)}, expected {out}")
    if out_dtype is not None and out_dtype != OUT_DTYPE[op]:
        raise ValueError(f"{op}: the output is {out_dtype}, expected {OUT_DTYPE[op]}")


def op_extras(op: str, shapes: list[tuple], attrs: dict) -> list[int]:
    """OpNode.extra of a cache op: [page_size, kv_heads, head_dim, type code, pages of the cache, pages of
    a table row, rows of the chunk (CACHE_WRITE), batch (CACHE_WRITE)]."""
    lay = CacheLayout.of(attrs)
    cache, table = (shapes[1], shapes[2]) if op == "PAGED_ATTENTION" else (shapes[0], shapes[-3])
    ex = [lay.page_size, lay.kv_heads, lay.head_dim, CACHE_TYPES[lay.cache_type][0], cache[0], table[1]]
    if op == "CACHE_WRITE":
        ex += [shapes[1][2], table[0]]
    return ex
