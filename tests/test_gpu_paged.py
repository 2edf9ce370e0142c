"""The paged-cache ops and VERIFY_DRAFT on the GPU against their definitions in 64 bits
(tests/paged_reference.py), alone and as a model uses them together."""

import numpy as np
import pytest
import torch   # before the library's first use, so that both take the same HIP runtime

from helpers import cf_attention, rng
from paged_reference import Pages, verify
from runtime.ir import Graph, OpType
from runtime.paged import CACHE_TYPES, CacheLayout
from runtime.session import Session

pytestmark = pytest.mark.gpu

TABLE = ["table", "start", "count"]


class Ops:
    """A graph over one cache; nodes are added, then it runs with the pages of a `Pages`."""

    def __init__(self, layout, pages):
        self.g, self.layout, self.feed = Graph(), layout, {}
        self.g.add_state("cache", layout.shape(pages.n))
        self.pages, self.at = pages, "cache"

    def input(self, name, value):
        if name not in self.feed:
            self.feed[name] = np.ascontiguousarray(value)
            self.g.add_tensor(name, value.shape, str(value.dtype))
            self.g.inputs.append(name)
        return name

    def where(self, table, start, count):
        for n, v in zip(TABLE, (table, start, count)):
            self.input(n, np.asarray(v, np.int32))
        return TABLE

    def write(self, k, v, *where):
        ins = [self.at, self.input("k", k), self.input("v", v), *self.where(*where)]
        self.at = "written"
        self.g.add_tensor(self.at, self.layout.shape(self.pages.n), "uint8")
        self.g.add_node(OpType.CACHE_WRITE, ins, self.at, self.layout.attrs)

    def attention(self, q, *where, **attrs):
        ins = [self.input("q", q), self.at, *self.where(*where)]
        self.g.add_tensor("y", q.shape)
        self.g.add_node(OpType.PAGED_ATTENTION, ins, "y", {**self.layout.attrs, **attrs})
        self.g.outputs.append("y")

    def read(self, length, *where):
        ins = [self.at, *self.where(*where)]
        lay = self.layout
        self.g.add_tensor("z", (2, len(where[1]), lay.kv_heads, length, lay.head_dim))
        self.g.add_node(OpType.CACHE_READ, ins, "z", {**lay.attrs, "length": length})
        self.g.outputs.append("z")

    def run(self, times=1):
        """(outputs, the cache's bytes after) of `times` runs, each the same."""
        s = Session(self.g)
        s.create()
        s.write_state("cache", self.pages.pack())
        try:
            out = s.run(self.feed)
            for _ in range(times - 1):
                for n, v in s.run(self.feed).items():
                    np.testing.assert_array_equal(v, out[n])
            return out, s.read_state("cache")
        finally:
            s.close()


def tables(r, batch, wide, n):
    """A page table of distinct pages among n."""
    return r.permutation(n)[:batch * wide].reshape(batch, wide).astype(np.int32)


def rows(r, *shape):
    return (r.standard_normal(shape) * np.exp(r.standard_normal((*shape[:-1], 1)))).astype(np.float32)


# ---------------------------------------------------------------- write and read

@pytest.mark.parametrize("kind", CACHE_TYPES)
@pytest.mark.parametrize("heads,hd,page,S,start,count", [
    (1, 64, 16, 1, [0, 5, 31], [1, 1, 0]),             # single tokens, one sequence without any
    (2, 128, 32, 21, [0, 3, 9], [21, 7, -2]),          # partial groups at both ends, a negative count
    (3, 24, 16, 8, [8, 16, 7], [8, 99, 2]),            # whole groups; more than the chunk holds
    (1, 1, 16, 17, [1, 30, 0], [17, 17, 17]),          # one column
    (2, 80, 64, 40, [60, 100, 24], [40, 40, 9]),       # across pages; past the table's end
    (1, 250, 16, 9, [-3, 2, 28], [9, 3, 9]),           # before position zero; head_dim no multiple of 4
    (1, 256, 128, 3, [0, 127, 255], [3, 3, 3]),
])
def test_write(kind, heads, hd, page, S, start, count):
    r = rng(heads * 1000 + hd + S)
    lay = CacheLayout(heads, hd, page, kind)
    table = tables(r, 3, 2, 9)
    table[0, 1] = -1
    table[1, 1] = 9          # pages the cache does not have
    pages = Pages.random(lay, 9, r)
    ops = Ops(lay, pages)
    k, v = rows(r, 3, heads, S, hd), rows(r, 3, heads, S, hd)
    ops.write(k, v, table, start, count)
    before = pages.pack()
    _, after = ops.run(times=2)
    pages.write(k, v, table, start, count)
    want = pages.pack()
    assert (want != before).any()
    np.testing.assert_array_equal(after, want)


@pytest.mark.parametrize("kind", CACHE_TYPES)
def test_write_special_rows(kind):
    """Infinities, NaN, zeros, subnormals, the largest values, and values next to a rounding's border."""
    r = rng(5)
    lay = CacheLayout(1, 64, 16, kind)
    S = 40
    k = rows(r, 1, 1, S, 64)
    k[0, 0, 0] = 0
    k[0, 0, 1, 3] = np.inf
    k[0, 0, 2, 60] = -np.inf
    k[0, 0, 3, 17] = np.nan
    k[0, 0, 4] = np.float32(1e-42) * np.arange(64)                 # subnormal throughout
    k[0, 0, 5] = r.standard_normal(64).astype(np.float32) * np.float32(2.0**-122)
    k[0, 0, 6] = r.uniform(-1, 1, 64).astype(np.float32) * np.float32(3.4e38)
    k[0, 0, 7, 0], k[0, 0, 7, 1:] = 3e38, np.float32(1e-12)
    k[0, 0, 8] = -0.0
    for i, top in ((9, 127.0), (10, 448.0), (11, 127.0 * 3)):       # exact ties, and their neighbours
        x = (np.arange(64) - 20.5).astype(np.float32) * np.float32(top / 127.0)
        k[0, 0, i], k[0, 0, i, 0] = x, top
        k[0, 0, i + 10], k[0, 0, i + 20] = np.nextafter(x, np.float32(1e9)), np.nextafter(x, np.float32(-1e9))
        k[0, 0, i + 10, 0] = k[0, 0, i + 20, 0] = top
    v = np.ascontiguousarray(k[:, :, ::-1])
    pages = Pages(lay, 4)
    ops = Ops(lay, pages)
    table = np.array([[3, 1, 0]], np.int32)
    ops.write(k, v, table, [2], [S])
    ops.read(S, table, [2], [S])
    out, after = ops.run()
    pages.write(k, v, table, [2], [S])
    np.testing.assert_array_equal(after, pages.pack())
    want = pages.read(table, [2], [S], S)
    np.testing.assert_array_equal(out["z"], want.astype(np.float32))
    for row in (1, 2, 3):
        assert np.isnan(out["z"][0, 0, 0, row]).all()


def test_write_borders_of_many_rows():
    """65536 values whose quotients lie on or next to a rounding's border: the scale is odd."""
    r = rng(11)
    for kind, top in (("int8", 127), ("float8", 448)):
        lay = CacheLayout(1, 256, 256, kind)
        k = np.zeros((1, 1, 256, 256), np.float32)
        for i in range(256):
            s = np.float32(np.float32(r.uniform(0.5, 2)) / 1)
            amax = np.float32(s * top)
            scale = np.float32(amax / np.float32(top))
            step = r.integers(-120, 120, 256) + 0.5 if kind == "int8" else \
                np.ldexp(r.integers(16, 32, 256) + 0.5, r.integers(-8, 3, 256))
            x = (step * float(scale)).astype(np.float32)
            k[0, 0, i] = np.where(r.random(256) < 0.5, x, np.nextafter(x, np.float32(r.choice([-1e9, 1e9]))))
            k[0, 0, i, 0] = amax
        pages = Pages(lay, 1)
        ops = Ops(lay, pages)
        where = (np.zeros((1, 1), np.int32), [0], [256])
        ops.write(k, k, *where)
        _, after = ops.run()
        pages.write(k, k, *where)
        np.testing.assert_array_equal(after, pages.pack())


@pytest.mark.parametrize("kind", CACHE_TYPES)
@pytest.mark.parametrize("heads,hd,page,T,start,count", [
    (1, 64, 16, 1, [0, 5, 31], [1, 1, 0]),
    (2, 128, 32, 50, [0, 3, 9], [50, 7, 0]),
    (3, 24, 16, 33, [8, 16, 7], [8, 99, -1]),          # rows past the table's end
    (1, 250, 16, 12, [-3, 2, 28], [9, 3, 9]),
    (2, 1, 64, 130, [0, 1, 2], [130, 127, 64]),
    (1, 256, 16, 20, [0, 12, 5], [20, 20, 20]),
])
def test_read(kind, heads, hd, page, T, start, count):
    r = rng(heads + hd + T)
    lay = CacheLayout(heads, hd, page, kind)
    table = tables(r, 3, 2, 8)
    table[2, 1] = 8
    pages = Pages.random(lay, 8, r)
    pages.s[table[0, 0], 0, 1, 7] = np.nan
    ops = Ops(lay, pages)
    ops.read(T, table, start, count)
    out, after = ops.run()
    np.testing.assert_array_equal(after, pages.pack())
    np.testing.assert_array_equal(out["z"], pages.read(table, start, count, T).astype(np.float32))


# ---------------------------------------------------------------- attention

ATTENTION = [
    # heads, kv_heads, head_dim, page, S, start, count, pages of a table row
    (1, 1, 64, 16, 1, [0], [1], 1),                              # one key
    (12, 12, 64, 16, 1, [36], [1], 3),
    (8, 2, 128, 32, 1, [0, 31, 32, 95], [1, 1, 1, 0], 3),        # page borders; a sequence without rows
    (32, 8, 128, 64, 1, [500, 3], [1, 1], 8),
    (4, 1, 80, 16, 5, [20, 7, 0], [5, 2, 0], 2),                 # drafted tokens
    (16, 2, 128, 16, 4, [130, 44], [4, 3], 9),                   # 32 rows a head
    (24, 2, 96, 16, 5, [40], [5], 3),                            # 60 rows
    (6, 2, 40, 16, 7, [10, 0], [7, 7], 2),
    (3, 3, 64, 16, 130, [0, 70], [130, 99], 13),                 # a first chunk; ragged
    (8, 2, 128, 32, 33, [65, 0], [33, 20], 4),
    (2, 2, 256, 16, 70, [3], [70], 5),
    (2, 1, 200, 64, 3, [300], [3], 5),
    (1, 1, 1, 16, 9, [5], [9], 1),
    (5, 5, 17, 16, 20, [11, 12], [20, 1], 2),
    (2, 2, 32, 128, 257, [0], [257], 3),
]


@pytest.mark.parametrize("kind", CACHE_TYPES)
@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: f"{c[0]}x{c[2]}_{c[4]}rows")
def test_attention(kind, case):
    H, kv, hd, page, S, start, count, wide = case
    r = rng(H + hd + S)
    lay = CacheLayout(kv, hd, page, kind)
    B = len(start)
    n = B * wide + 2
    pages = Pages.random(lay, n, r)
    table = tables(r, B, wide, n)
    q = 2 * r.standard_normal((B, H, S, hd)).astype(np.float32)
    ops = Ops(lay, pages)
    ops.attention(q, table, start, count)
    y = ops.run(times=3)[0]["y"]
    want, off = pages.attention(q, table, start, count)
    assert np.isfinite(want).all()
    assert (np.abs(y - want) <= off).all(), (np.abs(y - want).max(), off.max())
    assert np.linalg.norm(y - want) <= 2e-6 * np.linalg.norm(want) + 1e-30


@pytest.mark.parametrize("S", [1, 6, 40])
@pytest.mark.parametrize("kind", CACHE_TYPES)
def test_attention_nan_stays_with_the_rows_that_reach_it(kind, S):
    """A position with an infinity: rows before it are untouched, rows from it on are NaN; what lies behind
    a sequence's end, NaN patterns in every byte, reaches no row."""
    r = rng(S)
    lay = CacheLayout(1, 64, 16, kind)
    pages = Pages(lay, 8)
    k, v = rows(r, 1, 1, 10 + S, 64), rows(r, 1, 1, 10 + S, 64)
    at = 10 + S // 2
    (k if S == 6 else v)[0, 0, at, 5] = np.inf
    table = np.array([[5, 2, 7, 0]], np.int32)
    pages.write(k, v, table, [0], [10 + S])
    raw = pages.pack()
    garbage = np.full_like(raw, 0xff)
    part = 16 * 64 * CACHE_TYPES[kind][1]
    for pos in range(10 + S):                  # only written positions keep their bytes
        p, slot = table[0, pos // 16], pos % 16
        es = CACHE_TYPES[kind][1]
        for lo, hi in ((slot * 64 * es, (slot + 1) * 64 * es), (2 * part + 4 * slot, 2 * part + 4 * slot + 4),
                       (2 * part + 64 + 4 * slot, 2 * part + 64 + 4 * slot + 4)):
            garbage[p, lo:hi] = raw[p, lo:hi]
        va = garbage[p, part:2 * part].reshape(2, 64, 8, es)
        va[slot // 8, :, slot % 8] = raw[p, part:2 * part].reshape(2, 64, 8, es)[slot // 8, :, slot % 8]
    q = r.standard_normal((1, 4, S, 64)).astype(np.float32)
    ops = Ops(lay, pages)
    ops.attention(q, table, [10], [S])
    pages.pack = lambda: garbage
    y = ops.run()[0]["y"]
    want, off = Pages.attention(pages, q, table, [10], [S])
    rows_ = np.arange(S) + 10 < at
    assert np.isfinite(want[:, :, rows_]).all() and np.isnan(want[:, :, ~rows_]).all()
    assert np.isnan(y[:, :, ~rows_]).all()
    assert (np.abs(y - want) <= off)[:, :, rows_].all()


@pytest.mark.parametrize("S", [1, 9, 70])
def test_attention_bad_pages_and_positions(S):
    """Pages the cache does not have, a negative start and rows past the table give NaN, to the rows that
    reach them alone; counts past the chunk are the chunk."""
    r = rng(S + 1)
    lay = CacheLayout(2, 64, 16, "int8")
    pages = Pages.random(lay, 40, r)
    table = tables(r, 5, 7, 40)
    table[0, 0] = 40
    table[1, 1] = -7
    start = [5, 20, -1, 7 * 16 - S + 1, 3]
    count = [S, S, S, S, 1000]
    q = r.standard_normal((5, 4, S, 64)).astype(np.float32)
    ops = Ops(lay, pages)
    ops.attention(q, table, start, count)
    y = ops.run()[0]["y"]
    want, off = pages.attention(q, table, start, count)
    bad = np.isnan(want)
    assert bad[0].all() and bad[2].all() and bad[3, :, -1].all() and not bad[3, :, :-1].any() and not bad[4].any()
    np.testing.assert_array_equal(np.isnan(y), bad)
    assert (np.abs(y - want) <= off)[~bad].all()


@pytest.mark.parametrize("S", [1, 20])
def test_attention_of_large_and_tiny_rows(S):
    """Rows of 1e30 and 1e-30, peaked scores, and a scale of its own."""
    r = rng(2)
    for kind in CACHE_TYPES:
        lay = CacheLayout(1, 64, 16, kind)
        pages = Pages(lay, 6)
        k, v = rows(r, 1, 1, 60, 64), rows(r, 1, 1, 60, 64)
        k[0, 0, ::3] *= np.float32(1e-30)
        v[0, 0, ::2] *= np.float32(1e30)
        v[0, 0, 5] *= np.float32(1e-30)
        table = np.array([[4, 0, 2, 3]], np.int32)
        pages.write(k, v, table, [0], [60])
        q = 20 * r.standard_normal((1, 3, S, 64)).astype(np.float32)
        q[0, 1] *= np.float32(1e-25)
        q[0, 2] = 0
        ops = Ops(lay, pages)
        ops.attention(q, table, [60 - S], [S], scale=0.03)
        y = ops.run()[0]["y"]
        want, off = pages.attention(q, table, [60 - S], [S], scale=0.03)
        assert (np.abs(y - want) <= off).all()


def test_attention_scores_far_apart():
    """One key takes all the weight, first and last, against scores thousands below it."""
    r = rng(8)
    lay = CacheLayout(1, 64, 16, "float32")
    pages = Pages(lay, 40)
    k, v = rows(r, 1, 1, 600, 64), rows(r, 1, 1, 600, 64)
    table = tables(r, 1, 38, 40)
    q = r.standard_normal((1, 2, 1, 64)).astype(np.float32)
    k[0, 0, 3] = 800 * q[0, 0, 0]
    k[0, 0, 599] = 900 * q[0, 1, 0]
    pages.write(k, v, table, [0], [600])
    ops = Ops(lay, pages)
    ops.attention(q, table, [599], [1])
    y = ops.run()[0]["y"]
    np.testing.assert_allclose(y[0, 0, 0], v[0, 0, 3], rtol=1e-6)
    np.testing.assert_allclose(y[0, 1, 0], v[0, 0, 599], rtol=1e-6)


# ---------------------------------------------------------------- verification

def probabilities(r, *shape):
    x = np.exp(2 * r.standard_normal(shape))
    return (x / x.sum(-1, keepdims=True)).astype(np.float32)


def run_verify(*ins, times=1):
    g = Graph()
    feed = dict(zip(("target", "draft", "tokens", "uniforms", "count"), ins))
    for n, v in feed.items():
        g.add_tensor(n, v.shape, str(v.dtype))
        g.inputs.append(n)
    B, D = feed["tokens"].shape
    g.add_tensor("out", (B, D + 1), "int64")
    g.add_node(OpType.VERIFY_DRAFT, list(feed), "out")
    g.outputs.append("out")
    s = Session(g)
    s.create()
    try:
        out = s.run(feed)["out"]
        for _ in range(times - 1):
            np.testing.assert_array_equal(s.run(feed)["out"], out)
        return out
    finally:
        s.close()


@pytest.mark.parametrize("B,D,V", [(1, 0, 5), (3, 1, 1), (7, 4, 50), (40, 5, 5000), (5, 3, 4096), (4, 70, 130), (6, 2, 12289),
                                   (2, 8, 300001)])
def test_verify(B, D, V):
    r = rng(B + V)
    target = probabilities(r, B, D + 1, V)
    mix = 0.7 * target[:, :D].astype(np.float64) + 0.3 * probabilities(r, B, D, V)
    draft = mix.astype(np.float32)
    tokens = np.array([[r.choice(V, p=mix[b, i] / mix[b, i].sum()) for i in range(D)] for b in range(B)],
                      np.int64).reshape(B, D)
    uniforms = r.random((B, D + 1), dtype=np.float32)
    count = r.integers(0, D + 2, B).astype(np.int32)
    ins = (target, draft, tokens, uniforms, count)
    np.testing.assert_array_equal(run_verify(*ins, times=2), verify(*ins))


def test_verify_borders():
    """Equal rows, an exact tie, zeros, a mark at either end, numbers that are no probabilities, tokens
    outside the vocabulary."""
    V, D = 5000, 2
    p = np.zeros((12, D + 1, V), np.float32)
    q = np.zeros((12, D, V), np.float32)
    t = np.full((12, D), 7, np.int64)
    u = np.full((12, D + 1), 0.5, np.float32)
    p[:, :, 7], p[:, :, 4999], q[:, :, 7] = 0.25, 0.75, 0.5
    c = np.full(12, D, np.int32)
    # 0: u·q = p does not stand; the rest is all at 4999
    u[1, 0] = np.nextafter(np.float32(0.5), np.float32(0))      # 1: just stands, then falls
    q[2] = p[2, :D]
    u[2] = 0.999                                                # 2: equal rows: both stand, drawn from the target
    p[3, 0], q[3, 0] = 0, 0.5
    p[3, 0, 100] = 0.25                                         # 3: falls, nothing above the draft: the target's row
    p[4, 0] = 0                                                 # 4: nothing to draw from
    u[5, 2] = 1.0                                               # 5: a mark that no sum passes: the last entry
    u[6, 2] = 0.0
    p[6, 0, 40] = 1e-30                                         # 6: mark zero: the first entry above zero
    p[7, 0, 3], p[7, 0, 4500] = np.nan, np.inf                  # 7: NaN counts nothing, infinity everything
    p[8, 0, 3] = -1                                             # 8: nor does a negative one
    t[9, 0], t[10, 0] = -1, V                                   # 9, 10: no token of the vocabulary
    c[11] = 0                                                   # 11: nothing drafted
    out = run_verify(p, q, t, u, c)
    with np.errstate(invalid="ignore"):
        want = verify(p, q, t, u, c)
    np.testing.assert_array_equal(out[np.arange(12) != 7], want[np.arange(12) != 7])
    assert out[7, 0] in (4500, 4999) and (out[7, 1:] == -1).all()
    assert out[0].tolist() == [4999, -1, -1] and out[1].tolist() == [7, 4999, -1]
    assert out[2].tolist() == [7, 7, 4999] and out[3].tolist() == [100, -1, -1] and out[4].tolist() == [-1] * 3
    assert out[5, 0] == 4999 and out[6, 0] == 40 and out[11, 1] == -1


# ---------------------------------------------------------------- together

def step_session(layout, batch, heads, n_pages, wide, plan_cache=8, **device):
    """A layer's step, write then attend then read back, of a chunk of L tokens."""
    g = Graph()
    L = 4
    kv = (batch, layout.kv_heads, L, layout.head_dim)
    for name, shape, dtype in (("q", (batch, heads, L, layout.head_dim), "float32"), ("k", kv, "float32"),
                               ("v", kv, "float32"), ("table", (batch, wide), "int32"), ("start", (batch,), "int32"),
                               ("count", (batch,), "int32")):
        g.add_tensor(name, shape, dtype)
        g.inputs.append(name)
    g.add_state("cache", layout.shape(n_pages))
    g.add_tensor("written", layout.shape(n_pages), "uint8")
    g.add_tensor("y", (batch, heads, L, layout.head_dim))
    g.add_node(OpType.CACHE_WRITE, ["cache", "k", "v", *TABLE], "written", layout.attrs)
    g.add_node(OpType.PAGED_ATTENTION, ["q", "written", *TABLE], "y", layout.attrs)
    g.outputs.append("y")
    g.dynamic_dims = {"L": [("q", 2), ("k", 2), ("v", 2)]}
    s = Session(g)
    s.create(bindings={"L": L}, plan_cache=plan_cache, device_tensors=device or None)
    return s


@pytest.mark.parametrize("heads,kv,hd", [(4, 4, 64), (8, 2, 128)])
def test_chunks_equal_the_whole_sequence(heads, kv, hd):
    """Prompts of two lengths in chunks of several sizes, then single tokens: the dense attention of the whole
    sequences, over plans that share the cache."""
    r = rng(heads)
    lay = CacheLayout(kv, hd, 16, "float32")
    B, total = 2, [61, 47]
    x = [r.standard_normal((B, n, 61, hd)).astype(np.float32) for n in (heads, kv, kv)]
    table = tables(r, B, 4, 11)
    s = step_session(lay, B, heads, 11, 4)
    got = np.zeros((B, heads, 61, hd), np.float32)
    done = [0, 0]
    for L in (32, 17, 4, 1, 1, 1, 1, 4):
        s.rebind({"L": L})
        n = [min(L, total[b] - done[b]) for b in range(B)]
        feed = {name: np.zeros((B, a.shape[1], L, hd), np.float32) for name, a in zip("qkv", x)}
        for b in range(B):
            for name, a in zip("qkv", x):
                feed[name][b, :, :n[b]] = a[b, :, done[b]:done[b] + n[b]]
        y = s.run({**feed, "table": table, "start": np.array(done, np.int32), "count": np.array(n, np.int32)})["y"]
        for b in range(B):
            got[b, :, done[b]:done[b] + n[b]] = y[b, :, :n[b]]
            assert (y[b, :, n[b]:] == 0).all()
            done[b] += n[b]
    assert done == total and len(s.cached_plans) == 4
    for b in range(B):
        k, v = (np.repeat(a[b, :, :total[b]], heads // kv, 0) for a in x[1:])
        want = cf_attention(x[0][b, :, :total[b]], k, v, causal=True)
        assert np.abs(got[b, :, :total[b]] - want).max() <= 1e-5 * np.abs(want).max()
    before = s.read_state("cache")
    s.reset_states()
    assert before.any() and not s.read_state("cache").any()
    s.close()


def test_cache_and_inputs_in_the_callers_memory():
    """Inputs and the cache in torch tensors, outputs seen in place, work of torch's stream before and after;
    every replay against the definition."""
    r = rng(1)
    lay = CacheLayout(2, 64, 16, "float16")
    pages = Pages.random(lay, 9, r)
    table = tables(r, 2, 4, 9)
    q, k, v = (r.standard_normal((2, n, 4, 64)).astype(np.float32) for n in (4, 2, 2))
    dev = {"cache": torch.from_numpy(pages.pack()).cuda(), "table": torch.from_numpy(table).cuda(),
           "start": torch.tensor([17, 3], dtype=torch.int32, device="cuda"),
           "count": torch.tensor([4, 2], dtype=torch.int32, device="cuda")}
    dev |= {n: torch.empty(a.shape, device="cuda") for n, a in zip("qkv", (q, k, v))}
    torch.cuda.synchronize()
    s = step_session(lay, 2, 4, 9, 4, **dev)
    out = torch.as_tensor(s.device_outputs()["y"], device="cuda")
    host = [torch.from_numpy(a).cuda() for a in (q, k, v)]
    side = torch.cuda.Stream()
    for step in range(4):
        with torch.cuda.stream(side):
            for n, a in zip("qkv", host):
                dev[n].copy_(a * (step + 1))
            s.executor.wait_stream(side)
            s.executor.launch()
            s.executor.signal_stream(side)
            y = out.clone()
        side.synchronize()
        pages.write(k * np.float32(step + 1), v * np.float32(step + 1), table, [17, 3], [4, 2])
        want, off = pages.attention(q * np.float32(step + 1), table, [17, 3], [4, 2])
        assert (np.abs(y.cpu().numpy() - want) <= off).all()
        np.testing.assert_array_equal(dev["cache"].cpu().numpy(), pages.pack())
        torch.zeros(1 << 20, device="cuda").sum().item()   # work of the program's own between replays
    with pytest.raises(ValueError, match="caller's device memory"):
        s.run({"q": q, "k": k, "v": v})
    s.close()


def test_device_tensor_refusals():
    lay = CacheLayout(2, 64, 16, "float16")
    good = torch.zeros((2, 4, 4, 64), device="cuda")
    for bad, error in ((np.zeros((2, 4, 4, 64), np.float32), TypeError), (good[:1], ValueError), (good.double(), ValueError),
                       (good.transpose(0, 1).contiguous().transpose(0, 1), ValueError),
                       (torch.zeros(2 * 4 * 4 * 64 + 1, device="cuda")[1:].view(2, 4, 4, 64), ValueError)):
        with pytest.raises(error, match="device tensor 'q'"):
            step_session(lay, 2, 4, 9, 4, q=bad)
    with pytest.raises(ValueError, match="neither an input nor a state"):
        step_session(lay, 2, 4, 9, 4, w=good)


def test_two_sessions_share_a_cache():
    """Plans of two sessions over one cache in the caller's memory, launched in turn."""
    r = rng(4)
    lay = CacheLayout(1, 64, 16, "int8")
    cache = torch.zeros(lay.shape(8), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    a, b = (step_session(lay, 1, 1, 8, 4, cache=cache) for _ in range(2))
    pages = Pages(lay, 8)
    table = np.array([[6, 1, 3, 2]], np.int32)
    for step in range(4):
        q, k, v = (r.standard_normal((1, 1, 4, 64)).astype(np.float32) for _ in range(3))
        where = (table, np.array([4 * step], np.int32), np.array([4], np.int32))
        y = (a, b)[step % 2].run({"q": q, "k": k, "v": v, **dict(zip(TABLE, where))})["y"]
        pages.write(k, v, *where)
        want, off = pages.attention(q, *where)
        assert (np.abs(y - want) <= off).all()
    a.close()
    b.close()


def test_draft_and_verify_together():
    """A sequence continued by drafted tokens: attended as one chunk, verified, and the next call's start
    set from what stood; the positions given up are written over."""
    r = rng(9)
    lay = CacheLayout(1, 32, 16, "float32")
    V, D, hd = 40, 3, 32
    embed, head = r.standard_normal((V, hd)).astype(np.float32), r.standard_normal((hd, V)).astype(np.float32)
    s = step_session(lay, 1, 1, 6, 5)
    table = np.array([[4, 2, 0, 1, 5]], np.int32)

    def attend(tokens, start):
        s.rebind({"L": len(tokens)})
        e = embed[tokens][None, None]
        return s.run({"q": e, "k": e, "v": e, "table": table, "start": np.array([start], np.int32),
                      "count": np.array([len(tokens)], np.int32)})["y"][0, 0]

    def dense(tokens):
        e = embed[np.array(tokens)][None]
        return cf_attention(e, e, e, causal=True)[0]

    def probs(y):
        z = np.exp(0.3 * (y @ head))
        return (z / z.sum(-1, keepdims=True)).astype(np.float32)

    text = [3, 17, 8, 25]
    attend(text[:-1], 0)
    for _ in range(8):
        draft = probs(r.standard_normal((D, hd)))
        tokens = np.array([r.choice(V, p=d / d.sum()) for d in draft.astype(np.float64)])
        y = attend([text[-1], *tokens], len(text) - 1)
        want = dense(text + list(tokens))[len(text) - 1:]
        assert np.abs(y - want).max() <= 1e-5 * np.abs(want).max()
        ins = (probs(y)[None], draft[None], tokens[None].astype(np.int64), r.random((1, D + 1), dtype=np.float32),
               np.array([D], np.int32))
        out = run_verify(*ins)
        np.testing.assert_array_equal(out, verify(*ins))
        text += [int(t) for t in out[0] if t >= 0]
    s.close()
