"""The paged-cache ops on the GPU where sizes and uses are unusual: many sequences, shared pages, positions far away,
caches past 4 GiB, captured plans beside other work, the C entry points."""

import ctypes

import numpy as np
import pytest
import torch   # before the library's first use, so that both take the same HIP runtime

from helpers import rng
from paged_reference import Pages, verify
from runtime.ir import Graph, OpType
from runtime.paged import CACHE_TYPES, CacheLayout
from runtime.session import Session
from test_gpu_paged import TABLE, Ops, rows, run_verify, step_session, tables

pytestmark = pytest.mark.gpu


def check(y, pages, q, *where):
    want, off = pages.attention(q, *where)
    np.testing.assert_array_equal(np.isnan(y), np.isnan(want))
    ok = ~np.isnan(want)
    assert (np.abs(y - want)[ok] <= off[ok]).all(), np.nanmax(np.abs(y - want) - off)


@pytest.mark.parametrize("kind", ["float16", "int8"])
@pytest.mark.parametrize("S", [1, 18])
def test_many_sequences(kind, S):
    """Lines of more than 64 sequences with lengths from nothing to several steps, ranges that cross 64."""
    r = rng(S)
    B, wide = 150, 20
    lay = CacheLayout(2, 32, 16, kind)
    pages = Pages.random(lay, 40, r)
    table = r.integers(0, 40, (B, wide)).astype(np.int32)   # read only: sequences share pages
    start = r.integers(0, 60, B).astype(np.int32)
    start[[3, 63, 64, 70, 127, 128, 149]] = [290, 300, 299, 0, 260, 280, 299]
    count = r.integers(0, S + 1, B).astype(np.int32)
    count[[3, 64, 149]] = S
    q = r.standard_normal((B, 4, S, 32)).astype(np.float32)
    ops = Ops(lay, pages)
    ops.attention(q, table, start, count)
    out, after = ops.run(times=2)
    check(out["y"], pages, q, table, start, count)
    np.testing.assert_array_equal(after, pages.pack())


@pytest.mark.parametrize("S", [1, 40])
def test_pages_that_repeat(S):
    """A prefix that two sequences share, and one page twice in a row of the table."""
    r = rng(S)
    lay = CacheLayout(2, 64, 16, "float32")
    pages = Pages.random(lay, 8, r)
    table = np.array([[5, 2, 1, 0, 3, 6], [5, 2, 7, 7, 2, 4]], np.int32)
    where = (table, np.array([50, 47], np.int32), np.array([S, S], np.int32))
    q = r.standard_normal((2, 4, S, 64)).astype(np.float32)
    ops = Ops(lay, pages)
    ops.attention(q, *where)
    out, _ = ops.run()
    check(out["y"], pages, q, *where)


@pytest.mark.parametrize("kind", ["float16", "int8"])
@pytest.mark.parametrize("S", [1, 9, 70])
def test_starts_far_away(kind, S):
    """Starts and counts at the ends of their type: writes dropped, rows NaN, other sequences as ever."""
    r = rng(S)
    lay = CacheLayout(1, 64, 16, kind)
    pages = Pages.random(lay, 12, r)
    most, least = 2**31 - 1, -2**31
    table = tables(r, 2, 6, 12)[[0, 0, 0, 0, 0, 1]]
    start = np.array([most, least, most - S, 96, -1, 3], np.int32)
    count = np.array([S, S, most, S, least, most], np.int32)
    q, k, v = (r.standard_normal((6, h, S, 64)).astype(np.float32) for h in (2, 1, 1))
    ops = Ops(lay, pages)
    ops.write(k, v, table, start, count)
    ops.attention(q, table, start, count)
    ops.read(S, table, start, count)
    out, after = ops.run()
    pages.write(k, v, table, start, count)
    np.testing.assert_array_equal(after, pages.pack())
    np.testing.assert_array_equal(out["z"], pages.read(table, start, count, S).astype(np.float32))
    assert np.isnan(out["y"][:4]).all() and (out["y"][4] == 0).all()
    check(out["y"][5:], pages, q[5:], table[5:], start[5:], np.array([S], np.int32))


@pytest.mark.parametrize("rows_a_head", [32, 33])
@pytest.mark.parametrize("kind", CACHE_TYPES)
def test_both_kernels_at_their_border(kind, rows_a_head):
    r = rng(rows_a_head)
    lay = CacheLayout(2, 48, 32, kind)
    pages = Pages.random(lay, 20, r)
    table = tables(r, 2, 10, 20)
    q = r.standard_normal((2, 2, rows_a_head, 48)).astype(np.float32)
    where = (table, np.array([280, 0], np.int32), np.array([rows_a_head, rows_a_head - 1], np.int32))
    ops = Ops(lay, pages)
    ops.attention(q, *where)
    check(ops.run()[0]["y"], pages, q, *where)


@pytest.mark.parametrize("S", [1, 20])
def test_cache_past_four_gigabytes(S):
    """Pages whose bytes lie behind 2^32, written, attended and read."""
    r = rng(S)
    lay = CacheLayout(2, 64, 1024, "float32")
    n = (1 << 32) // lay.page_bytes + 3
    pages = Pages.random(lay, 3, r)
    at = np.array([n - 1, 7, n - 2])                       # where the three lie
    cache = torch.zeros(lay.shape(n), dtype=torch.uint8, device="cuda")
    cache[torch.from_numpy(at).cuda()] = torch.from_numpy(pages.pack()).cuda()
    torch.cuda.synchronize()
    table, start, count = np.array([[0, 1, 2]], np.int32), np.array([2040], np.int32), np.array([S], np.int32)
    q, k, v = (r.standard_normal((1, h, S, 64)).astype(np.float32) for h in (4, 2, 2))
    g = Ops(lay, Pages(lay, 1))
    g.g.tensors["cache"].shape = lay.shape(n)
    g.pages.n = n
    there = at[table].astype(np.int32)
    g.write(k, v, there, start, count)
    g.attention(q, there, start, count)
    g.read(S, there, start, count)
    s = Session(g.g)
    s.create(device_tensors={"cache": cache})
    out = s.run(g.feed)
    pages.write(k, v, table, start, count)
    check(out["y"], pages, q, table, start, count)
    np.testing.assert_array_equal(out["z"], pages.read(table, start, count, S).astype(np.float32))
    np.testing.assert_array_equal(cache[torch.from_numpy(at).cuda()].cpu().numpy(), pages.pack())
    assert int(cache[:7].sum()) == int(cache[8:n - 2].any()) == 0
    s.close()


def layers_session(lay, n, B, H, S, wide, layers=2, **device):
    """Several layers' steps, each with a cache of its own, attention feeding the next layer's queries."""
    g = Graph()
    kv = (B, lay.kv_heads, S, lay.head_dim)
    for name, shape, dtype in (("q", (B, H, S, lay.head_dim), "float32"), ("k", kv, "float32"), ("v", kv, "float32"),
                               ("table", (B, wide), "int32"), ("start", (B,), "int32"), ("count", (B,), "int32")):
        g.add_tensor(name, shape, dtype)
        g.inputs.append(name)
    at = "q"
    for i in range(layers):
        g.add_state(f"cache{i}", lay.shape(n))
        g.add_tensor(f"written{i}", lay.shape(n), "uint8")
        g.add_node(OpType.CACHE_WRITE, [f"cache{i}", "k", "v", *TABLE], f"written{i}", lay.attrs)
        g.add_tensor(f"y{i}", (B, H, S, lay.head_dim))
        g.add_node(OpType.PAGED_ATTENTION, [at, f"written{i}", *TABLE], f"y{i}", lay.attrs)
        at = f"y{i}"
    g.add_tensor("z", (2, B, lay.kv_heads, 64, lay.head_dim))
    g.add_node(OpType.CACHE_READ, ["written0", *TABLE], "z", {**lay.attrs, "length": 64})
    g.outputs = [at, "z"]
    g.dynamic_dims = {"L": [("q", 2), ("k", 2), ("v", 2)]}
    s = Session(g)
    s.create(bindings={"L": S}, device_tensors=device or None)
    return s


@pytest.mark.parametrize("kind", ["float32", "int8"])
def test_captured_plans_in_turn(kind):
    """Plans of more than three kernel steps, captured: two of one session, whose caches are the same, and one of
    another session, replayed in turn with the program's own work between, each replay against the definition."""
    r = rng(3)
    B, H, wide, n = 2, 4, 30, 61
    lay = CacheLayout(2, 32, 16, kind)
    table = tables(r, B, wide, n)
    a, b = layers_session(lay, n, B, H, 1, wide), layers_session(lay, n, B, H, 40, wide)
    held = {id(s): [Pages(lay, n), Pages(lay, n)] for s in (a, b)}
    at = {id(s): np.array([0, 0]) for s in (a, b)}
    for s, S in ((a, 40), (b, 40), (a, 1), (a, 1), (b, 40), (b, 1), (a, 40), (a, 1), (b, 1), (a, 1)):
        s.rebind({"L": S})
        q, k, v = (r.standard_normal((B, h, S, 32)).astype(np.float32) for h in (H, 2, 2))
        count = np.array([S, max(1, S - 3)], np.int32)
        where = (table, at[id(s)].astype(np.int32), count)
        out = s.run({"q": q, "k": k, "v": v, **dict(zip(TABLE, where))})
        torch.zeros(1 << 20, device="cuda").sum().item()
        for p in held[id(s)]:
            p.write(k, v, *where)
        first, off = held[id(s)][0].attention(q, *where)
        want, own = held[id(s)][1].attention(first, *where)
        # an error d of a layer's queries moves its scores by at most |d| times the largest K row, and an output by
        # twice that of the largest V
        big = [np.nanmax(np.abs(held[id(s)][1].rows(table, i, h, j, range(int(where[1][i] + count[i]))))) for j in (0, 1)
               for i in range(B) for h in range(2)]
        slack = 2 * off.max() * np.sqrt(32) * max(big[:4]) * max(big[4:])
        assert (np.abs(out["y1"] - want) <= own + slack).all()
        np.testing.assert_array_equal(out["z"], held[id(s)][0].read(*where, 64).astype(np.float32))
        for i, p in enumerate(held[id(s)]):
            np.testing.assert_array_equal(s.read_state(f"cache{i}"), p.pack())
        at[id(s)] = at[id(s)] + count
    a.close()
    b.close()


def test_profiled_run_gives_the_same():
    r = rng(5)
    lay = CacheLayout(2, 64, 16, "float16")
    s = step_session(lay, 2, 4, 9, 4)
    feed = {n: r.standard_normal((2, h, 4, 64)).astype(np.float32) for n, h in (("q", 4), ("k", 2), ("v", 2))}
    feed |= dict(zip(TABLE, (tables(r, 2, 4, 9), np.array([17, 3], np.int32), np.array([4, 2], np.int32))))
    y = s.run(feed)["y"]
    np.testing.assert_array_equal(s.run(feed, profile=True)["y"], y)   # the same rows are written again
    assert s.last_profile is not None
    s.close()


def test_sequences_without_rows():
    """No sequence has rows in the call: outputs are zeros and the cache stays."""
    r = rng(6)
    lay = CacheLayout(2, 64, 16, "int8")
    pages = Pages.random(lay, 9, r)
    table, start, count = tables(r, 2, 4, 9), np.array([17, 0], np.int32), np.array([0, -5], np.int32)
    for S in (1, 50):
        q, k, v = (r.standard_normal((2, h, S, 64)).astype(np.float32) for h in (4, 2, 2))
        ops = Ops(lay, pages)
        ops.write(k, v, table, start, count)
        ops.attention(q, table, start, count)
        ops.read(7, table, start, count)
        out, after = ops.run()
        assert (out["y"] == 0).all() and (out["z"] == 0).all()
        np.testing.assert_array_equal(after, pages.pack())


@pytest.mark.parametrize("S", [2, 48])
@pytest.mark.parametrize("entry", ["lbr_execute", "lbr_execute_noalloc"])
def test_c_entry_points(hip_lib, entry, S):
    """The node array through the C ABI's one-shot entries gives what the plan gives."""
    from runtime.executor.compiled import CompiledExecutor, DeviceStates
    from runtime.planner import plan
    r = rng(S)
    lay = CacheLayout(2, 64, 16, "float16")
    pages = Pages.random(lay, 40, r)
    ops = Ops(lay, pages)
    where = (tables(r, 2, 20, 40), np.array([250, 3], np.int32), np.array([S, S - 1], np.int32))
    q, k, v = (rows(r, 2, h, S, 64) for h in (4, 2, 2))
    ops.write(k, v, *where)
    ops.attention(q, *where)
    ex = CompiledExecutor(fuse=False, states=DeviceStates(hip_lib))
    ex.compile(plan(ops.g))
    ex.write_state("cache", pages.pack())
    y = ex.run(ops.feed)["y"]
    after = ex.read_state("cache")
    ex.write_state("cache", pages.pack())
    hip_lib.lbr_memset(ctypes.c_void_p(ex.device_address("y")), 0, y.nbytes)
    ex.upload_inputs(ops.feed)
    hip_lib.check(getattr(hip_lib, entry)(ex._nodes, len(ex.dispatch_order)), entry)
    np.testing.assert_array_equal(ex.download_outputs()["y"], y)
    np.testing.assert_array_equal(ex.read_state("cache"), after)
    pages.write(k, v, *where)
    check(y, pages, q, *where)
    ex.close()


@pytest.mark.parametrize("B,S,T", [(2, 0, 3), (2, 1, 0), (0, 3, 3), (0, 0, 0)])
def test_sizes_of_zero(B, S, T):
    r = rng(1)
    lay = CacheLayout(2, 64, 16, "int8")
    pages = Pages.random(lay, 9, r)
    where = (tables(r, B, 4, 9), np.full(B, 5, np.int32), np.full(B, S, np.int32))
    q, k, v = (np.zeros((B, h, S, 64), np.float32) for h in (4, 2, 2))
    ops = Ops(lay, pages)
    ops.write(k, v, *where)
    ops.attention(q, *where)
    ops.read(T, *where)
    out, after = ops.run()
    pages.write(k, v, *where)
    assert out["y"].shape == (B, 4, S, 64)
    np.testing.assert_array_equal(out["z"], pages.read(*where, T).astype(np.float32))
    np.testing.assert_array_equal(after, pages.pack())


@pytest.mark.parametrize("B,D", [(0, 3), (2, 0), (0, 0)])
def test_verify_of_nothing(B, D):
    r = rng(2)
    p = r.dirichlet(np.ones(7), (B, D + 1)).astype(np.float32).reshape(B, D + 1, 7)
    ins = (p, np.zeros((B, D, 7), np.float32), np.zeros((B, D), np.int64), r.random((B, D + 1), dtype=np.float32),
           np.zeros(B, np.int32))
    np.testing.assert_array_equal(run_verify(*ins), verify(*ins))
