"""The paged-cache ops as torch ops and through the exporter, and models that continue their sequences."""

import numpy as np
import pytest
import torch

import workloads as wl
from conftest import normwise_rel
from paged_reference import Pages, verify
from runtime.exporter import export_model
from runtime.ir import Graph, OpType
from runtime.ops import resolve_graph
from runtime.paged import CACHE_TYPES, CacheLayout
from runtime.passes.passes import run_pipeline
from runtime.planner import plan
from runtime.validation import Phase, run_validators
from runtime.validation.core import ValidationError

lbr = torch.ops.lbr


def t(*arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)) for a in arrays]


# ---------------------------------------------------------------- the torch ops against the definitions

def example(kind, S=5, hd=24, page=16, seed=0):
    """A cache of rows, and a ragged chunk whose table holds pages that are none and ends inside the chunk."""
    r = np.random.default_rng(seed)
    lay = CacheLayout(2, hd, page, kind)
    pages = Pages.random(lay, 9, r)
    table = r.permutation(9)[:8].reshape(4, 2).astype(np.int32)
    table[2, 1] = 9
    start, count = np.array([0, 14, 13, 30], np.int32), np.array([S, 3, S, S], np.int32)
    k, v = (r.standard_normal((4, 2, S, hd)).astype(np.float32) for _ in range(2))
    k[0, 1, 2, 3], v[1, 0, 0, 0], k[3, 0, 0] = np.inf, np.nan, 0.0
    return r, lay, pages, table, start, count, k, v


@pytest.mark.parametrize("kind", CACHE_TYPES)
def test_torch_write_and_read(kind):
    _, lay, pages, table, start, count, k, v = example(kind)
    cache = torch.from_numpy(pages.pack())
    lbr.cache_write(cache, *t(k, v, table, start, count), lay.page_size, kind)
    pages.write(k, v, table, start, count)
    np.testing.assert_array_equal(cache.numpy(), pages.pack())
    got = lbr.cache_read(cache, *t(table, start - 2, count), 4, lay.kv_heads, lay.head_dim, lay.page_size, kind)
    np.testing.assert_array_equal(got.numpy(), pages.read(table, start - 2, count, 4).astype(np.float32))


@pytest.mark.parametrize("kind", CACHE_TYPES)
@pytest.mark.parametrize("scale", [None, 0.3])
def test_torch_attention(kind, scale):
    r, lay, pages, table, start, count, k, v = example(kind)
    pages.write(k, v, table, start, count)
    q = r.standard_normal((4, 6, 5, lay.head_dim)).astype(np.float32)
    start[0] = -1
    want, _ = pages.attention(q, table, start, count, scale)
    got = lbr.paged_attention(*t(q, pages.pack(), table, start, count), lay.kv_heads, lay.page_size, kind, scale).numpy()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    # both in 64 bits, one rounded to 32 at the end
    np.testing.assert_allclose(got, want, rtol=2.0**-23, atol=1e-12)


def test_torch_verify():
    r = np.random.default_rng(2)
    p = r.dirichlet(np.ones(9), (40, 4)).astype(np.float32)
    q = r.dirichlet(np.ones(9), (40, 3)).astype(np.float32)
    p[0], q[1], p[2, 0] = 0, p[1, :3], np.nan
    tokens = r.integers(-1, 10, (40, 3))
    u, count = r.random((40, 4)).astype(np.float32), r.integers(-1, 5, 40).astype(np.int32)
    np.testing.assert_array_equal(lbr.verify_draft(*t(p, q, tokens, u, count)).numpy(), verify(p, q, tokens, u, count))


def test_torch_op_refusals():
    _, lay, pages, table, start, count, k, v = example("int8")
    cache, k, v, table, start, count = t(pages.pack(), k, v, table, start, count)
    with pytest.raises(ValueError, match="page_size"):
        lbr.cache_write(cache, k, v, table, start, count, 24, "int8")
    with pytest.raises(ValueError, match="bytes"):
        lbr.cache_write(cache, k, v, table, start, count, 16, "float16")
    with pytest.raises(ValueError, match="start"):
        lbr.cache_read(cache, table, start.long(), count, 4, 2, 24, 16, "int8")
    with pytest.raises(ValueError, match="query heads"):
        lbr.paged_attention(torch.zeros(4, 3, 5, 24), cache, table, start, count, 2, 16, "int8")
    with pytest.raises(ValueError, match="target"):
        lbr.verify_draft(torch.zeros(2, 3, 9), torch.zeros(2, 3, 9), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 4),
                         torch.zeros(2, dtype=torch.int32))


# ---------------------------------------------------------------- the models

def index(*values):
    return np.array(values, np.int32)


def block(kind="float32", kv_heads=None, seed=3):
    m = wl.init_weights(wl.CachedGeluBlock(64, 4, 12, 16, kind, kv_heads=kv_heads), seed)
    with torch.no_grad():   # larger scores than 0.02-weights give
        m.wq.weight *= 12
        m.wk.weight *= 12
    return m


def whole(m, x):
    """The same block over whole sequences, without a cache, in 64 bits."""
    plain = wl.CausalGeluBlock(64, 4)
    state = {k: v for k, v in m.state_dict().items() if k != "cache"}
    plain.load_state_dict(state)
    with torch.no_grad():
        return plain.double()(torch.from_numpy(x).double()).numpy()


def test_chunks_of_a_model_equal_the_whole_sequence():
    m = block()
    x = np.random.default_rng(0).standard_normal((2, 60, 64)).astype(np.float32)
    table = np.random.default_rng(1).permutation(12)[:8].reshape(2, 4).astype(np.int32)
    want = whole(m, x)
    with torch.no_grad():
        m = m.double()
        for at, end in ((0, 33), (33, 34), (34, 60)):
            got = m(torch.from_numpy(x[:, at:end]).double(), *t(table, index(at, at), index(end - at, end - at)))
            # K and V are rounded to 32 bits: scores of up to 30 off by 2^-24 of themselves
            assert normwise_rel(got.numpy(), want[:, at:end]) < 60 * 2.0**-24


def exported(m, S=5, **dynamic):
    start, count = (torch.zeros(3, dtype=torch.int32) for _ in range(2))
    return export_model(m, (torch.zeros(3, S, 64), torch.zeros(3, 4, dtype=torch.int32), start, count), dynamic or None)


def test_export_makes_the_buffer_a_state():
    g = exported(block("int8"))
    assert g.states == ["b_cache"] and "b_cache" not in g.constants and g.tensors["b_cache"].buffer is None
    ops = [n.op for n in g]
    assert ops.count(OpType.CACHE_WRITE) == 1 and ops.index(OpType.CACHE_WRITE) < ops.index(OpType.PAGED_ATTENTION)
    write, = (n for n in g if n.op == OpType.CACHE_WRITE)
    attend, = (n for n in g if n.op == OpType.PAGED_ATTENTION)
    assert attend.inputs[1] == write.output and write.attrs == CacheLayout(4, 16, 16, "int8").attrs
    run_pipeline(g)
    mem = plan(g)
    assert OpType.CACHE_WRITE in [n.op for n in mem.order]


def test_export_copies_what_the_cache_holds():
    m = block("int8")
    m.cache[1, 2] = 7
    g = exported(m)
    m.cache[1, 2] = 9
    assert g.tensors["b_cache"].buffer[1, 2] == 7


def test_export_of_any_chunk_length(tmp_path):
    g = exported(block(), L=[("x", 1)])
    attend, = (n for n in g if n.op == OpType.PAGED_ATTENTION)
    assert attend.inputs[3:] == ["start", "count"]
    for length in (1, 3, 40):
        r = resolve_graph(g, {"L": length})
        assert r.tensors[attend.output].shape == (3, 4, length, 16)
        plan(r)
    r.save(tmp_path / "g.json")
    assert Graph.load(tmp_path / "g.json").states == ["b_cache"]


class Twice(torch.nn.Module):
    """Two writes of a cache, attention behind them; `before`: a reading ahead of them."""

    def __init__(self, before):
        super().__init__()
        self.before = before
        self.register_buffer("cache", torch.zeros(CacheLayout(2, 24, 16).shape(4), dtype=torch.uint8))

    def forward(self, k, table, start, count):
        out = [lbr.cache_read(self.cache, table, start, count, 5, 2, 24, 16, "float32")] if self.before else []
        lbr.cache_write(self.cache, k, k, table, start, count, 16, "float32")
        lbr.cache_write(self.cache, k + 1, k, table, start, count, 16, "float32")
        return *out, lbr.paged_attention(k, self.cache, table, start, count, 2, 16, "float32", scale=0.25)


def export_twice(before):
    return export_model(Twice(before), (torch.zeros(2, 2, 5, 24), torch.zeros(2, 2, dtype=torch.int32),
                                        *(torch.zeros(2, dtype=torch.int32) for _ in range(2))))


def test_export_reads_what_was_written_last():
    g = export_twice(False)
    first, second = (n for n in g if n.op == OpType.CACHE_WRITE)
    attend, = (n for n in g if n.op == OpType.PAGED_ATTENTION)
    assert first.inputs[0] == "b_cache" and second.inputs[0] == first.output
    assert attend.inputs[1] == second.output and attend.attrs["scale"] == 0.25
    assert not run_validators(Phase.POST_OPTIMIZE, g)
    plan(g)


def test_a_reading_ahead_of_a_write_is_refused():
    """Nothing in a graph orders the two."""
    with pytest.raises(ValidationError, match="uses the value before"):
        run_validators(Phase.POST_OPTIMIZE, export_twice(True))


def test_export_refuses_a_cache_that_is_an_input():
    class Input(torch.nn.Module):
        def forward(self, cache, k, table, start):
            lbr.cache_write(cache, k, k, table, start, start, 16, "float32")
            return k + 1

    with pytest.raises(ValueError, match="not a buffer of the model"):
        export_model(Input(), (torch.zeros(CacheLayout(2, 24, 16).shape(4), dtype=torch.uint8), torch.zeros(2, 2, 5, 24),
                               torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)))


# ---------------------------------------------------------------- on the device

@pytest.mark.gpu
@pytest.mark.parametrize("kind,kv_heads", [("float32", None), ("float16", 2)])
@pytest.mark.parametrize("optimization", ["default", "none"])
def test_model_in_chunks(hip_lib, kind, kv_heads, optimization):
    from runtime.session import Session
    m = block(kind, kv_heads)
    r = np.random.default_rng(5)
    table = r.permutation(12).reshape(3, 4).astype(np.int32)
    s = Session(exported(m, L=[("x", 1)]))
    s.create(bindings={"L": 1}, optimization=optimization)
    m = m.double()
    at = np.zeros(3, np.int32)
    for length in (20, 1, 1, 7, 1, 9):   # ragged: not every sequence fills the chunk
        x = r.standard_normal((3, length, 64)).astype(np.float32)
        count = np.minimum(length, index(length, max(1, length - 2), 1))
        s.rebind({"L": length})
        got, = s.run({"x": x, "page_table": table, "start": at, "count": count}).values()
        with torch.no_grad():
            want = m(torch.from_numpy(x).double(), *t(table, at, count)).numpy()
        for b in range(3):
            assert normwise_rel(got[b, :count[b]], want[b, :count[b]]) < 1e-3
        at = (at + count).astype(np.int32)
    s.close()


def language_model(seed, pages=18, n_layer=2, kind="float16"):
    m = wl.init_weights(wl.CachedLM(61, n_layer, 4, 64, 96, pages, 16, kind, kv_heads=2), seed)
    with torch.no_grad():
        m.wte.weight *= 20
        m.wpe.weight *= 10
    return m


def eager(m, tokens):
    """Probabilities behind the last token of one sequence, from a cache of its own."""
    ids = torch.tensor([tokens])
    with torch.no_grad():
        m.double()
        for b in m.h:
            b.cache.zero_()
        one = torch.zeros(1, dtype=torch.int32)
        table = torch.arange(m.h[0].cache.shape[0], dtype=torch.int32)[None]
        p = m(ids, torch.arange(len(tokens))[None], table, one, one + len(tokens))
    return p[0, -1].numpy()


PROMPTS = [[3, 7, 11], [5], list(range(20))]


def check_caches(gen, m, prompts, out):
    """The target's cache holds what the sequences are: the next probabilities are those of a fresh run."""
    seqs = [p + o for p, o in zip(prompts, out)]
    start = np.array([len(s) - 1 for s in seqs])
    p = gen.step(gen.target, np.array([[s[-1]] for s in seqs]), start, np.ones(len(seqs), np.int64))
    for b, s in enumerate(seqs):
        assert normwise_rel(p[b, 0], eager(m, s)) < 1e-3


@pytest.mark.gpu
def test_generate_token_by_token(hip_lib):
    m = language_model(1)
    gen = wl.Generator(m, 3)
    out = gen.generate(PROMPTS, 30, seed=4)
    assert [len(o) for o in out] == [30] * 3 and all(0 <= x < 61 for o in out for x in o)
    check_caches(gen, m, PROMPTS, out)
    assert gen.generate(PROMPTS, 30, seed=4) == out   # behind what the first run left in the pages


@pytest.mark.gpu
@pytest.mark.parametrize("draft_seed", [1, 2])
def test_generate_with_drafts(hip_lib, draft_seed):
    """A drafting model of the target's own weights, whose tokens stand, and another one."""
    m = language_model(1)
    gen = wl.Generator(m, 3, draft=language_model(draft_seed), drafts=4)
    out = gen.generate(PROMPTS, 30, seed=4)
    assert [len(o) for o in out] == [30] * 3 and all(0 <= x < 61 for o in out for x in o)
    check_caches(gen, m, PROMPTS, out)
    assert gen.generate(PROMPTS, 30, seed=4) == out


def test_generator_refusals(monkeypatch):
    monkeypatch.setattr(wl.Generator, "_create", lambda *a, **k: None)
    m = language_model(1)
    with pytest.raises(ValueError, match="too small"):
        wl.Generator(m, 19)
    for batch, drafts in ((0, 3), (3, 0)):
        with pytest.raises(ValueError, match="drafted tokens"):
            wl.Generator(m, batch, drafts=drafts)
    with pytest.raises(ValueError, match="drafting model"):
        wl.Generator(m, 3, draft=language_model(1, pages=17))
    gen = wl.Generator(m, 3)
    with pytest.raises(ValueError, match="prompts"):
        gen.generate(PROMPTS[:2], 4)
    with pytest.raises(ValueError, match="prompts"):
        gen.generate([*PROMPTS[:2], []], 4)
    with pytest.raises(ValueError, match="do not fit"):
        gen.generate(PROMPTS, 77)
    assert gen.generate(PROMPTS, 0) == [[], [], []]
