"""The paged-cache ops on the CPU: layouts, refusals, planning, the state rules, the library's own
checks of malformed records, and the reference that the device tests compare with."""

import ctypes

import numpy as np
import pytest

from paged_reference import Pages, e4m3_table, row_scale, store
from runtime.executor.common import COpNode
from runtime.executor.hip_lib import HipExecutorError, open_library
from runtime.executor.nodes import build_nodes, check_extents, dispatch_order
from runtime.ir import Graph, OpType
from runtime.paged import CACHE_TYPES, CacheLayout, check_op
from runtime.passes.passes import run_pipeline
from runtime.planner import plan
from runtime.validation import Phase, run_validators

LAY = CacheLayout(2, 24, 16, "int8")


def _tensor(g, name, shape, dtype="float32", role="inputs"):
    g.add_tensor(name, shape, dtype)
    if role:
        getattr(g, role).append(name)
    return name


def step_graph(layout=LAY, batch=3, heads=4, chunk=5, pages=7, wide=2, read=0):
    """One layer's step: write the chunk, attend, and with `read` read that many positions back."""
    g = Graph()
    kv = (batch, layout.kv_heads, chunk, layout.head_dim)
    _tensor(g, "q", (batch, heads, chunk, layout.head_dim))
    _tensor(g, "k", kv)
    _tensor(g, "v", kv)
    _tensor(g, "table", (batch, wide), "int32")
    _tensor(g, "start", (batch,), "int32")
    _tensor(g, "count", (batch,), "int32")
    g.add_state("cache", layout.shape(pages))
    _tensor(g, "cache2", layout.shape(pages), "uint8", None)
    g.add_node(OpType.CACHE_WRITE, ["cache", "k", "v", "table", "start", "count"], "cache2", layout.attrs)
    _tensor(g, "y", (batch, heads, chunk, layout.head_dim), role="outputs")
    g.add_node(OpType.PAGED_ATTENTION, ["q", "cache2", "table", "start", "count"], "y", layout.attrs)
    if read:
        _tensor(g, "z", (2, batch, layout.kv_heads, read, layout.head_dim), role="outputs")
        g.add_node(OpType.CACHE_READ, ["cache2", "table", "start", "count"], "z", {**layout.attrs, "length": read})
    return g


def host_nodes(g):
    """The node array over made-up aligned addresses, and its live ranges."""
    mem = plan(g)
    at, addr = 1 << 20, {}
    for n in g.tensors:
        addr[n], at = at, at + (1 << 20)
    for node in g.nodes.values():
        if node.op == OpType.CACHE_WRITE:
            addr[node.output] = addr[g.state_of(node.output)]
    return build_nodes(mem, addr.__getitem__, lambda off, size: at + off)


@pytest.mark.parametrize("kind", CACHE_TYPES)
@pytest.mark.parametrize("heads,hd,page", [(1, 1, 16), (5, 80, 64), (8, 128, 128), (3, 255, 32768 // 64)])
def test_layout_sizes(kind, heads, hd, page):
    lay = CacheLayout(heads, hd, page, kind)
    es = CACHE_TYPES[kind][1]
    assert lay.row % 16 == 0 and 0 <= lay.row - hd < 16
    assert lay.page_bytes == heads * page * (2 * lay.row * es + 8)
    assert lay.shape(9) == (9, lay.page_bytes) and lay.head_bytes % 16 == 0
    assert CacheLayout.of(lay.attrs) == lay


@pytest.mark.parametrize("args", [(0, 64, 16, "int8"), (1, 0, 16, "int8"), (1, 257, 16, "int8"), (1, 64, 8, "int8"),
                                  (1, 64, 48, "int8"), (1, 64, 65536, "int8"), (1, 64, 16, "int4"),
                                  (1 << 14, 256, 1024, "float32")])
def test_layout_refusals(args):
    with pytest.raises(ValueError):
        CacheLayout(*args)


def _case(op):
    table = [((3, 2), "int32"), ((3,), "int32"), ((3,), "int32")]
    cache = (LAY.shape(7), "uint8")
    q, kv = ((3, 4, 5, 24), "float32"), ((3, 2, 5, 24), "float32")
    return {"CACHE_WRITE": [cache, kv, kv, *table], "CACHE_READ": [cache, *table], "PAGED_ATTENTION": [q, cache, *table],
            "VERIFY_DRAFT": [((2, 4, 9), "float32"), ((2, 3, 9), "float32"), ((2, 3), "int64"), ((2, 4), "float32"),
                             ((2,), "int32")]}[op]


def _attrs(op):
    return {} if op == "VERIFY_DRAFT" else {**LAY.attrs, **({"length": 6} if op == "CACHE_READ" else {})}


@pytest.mark.parametrize("op", ["CACHE_WRITE", "CACHE_READ", "PAGED_ATTENTION", "VERIFY_DRAFT"])
def test_op_refusals(op):
    good = _case(op)
    check_op(op, [s for s, _ in good], [d for _, d in good], _attrs(op))
    for k in range(len(good)):
        shapes, dtypes = [s for s, _ in good], [d for _, d in good]
        with pytest.raises(ValueError, match="expected"):   # a wrong type
            check_op(op, shapes, dtypes[:k] + ["float64"] + dtypes[k + 1:], _attrs(op))
        for d in range(len(shapes[k])):                     # every dim one too large
            if op == "PAGED_ATTENTION" and k == 0 and d in (1, 2):
                continue                                    # another number of heads or rows: allowed or below
            if (op, k, d) in (("CACHE_WRITE", 0, 0), ("CACHE_READ", 0, 0), ("PAGED_ATTENTION", 1, 0)):
                continue                                    # pages of the cache
            if (op != "VERIFY_DRAFT" and k == len(good) - 3 and d == 1):
                continue                                    # pages of a table row
            s = list(shapes[k])
            s[d] += 1
            with pytest.raises(ValueError):
                check_op(op, shapes[:k] + [tuple(s)] + shapes[k + 1:], dtypes, _attrs(op))
    with pytest.raises(ValueError, match="takes"):
        check_op(op, shapes[:-1], dtypes[:-1], _attrs(op))
    if op == "PAGED_ATTENTION":
        with pytest.raises(ValueError, match="query heads"):
            check_op(op, [(3, 5, 5, 24), *shapes[1:]], dtypes, _attrs(op))
        for scale in (0.0, -1.0, float("inf"), float("nan")):
            with pytest.raises(ValueError, match="scale"):
                check_op(op, shapes, dtypes, {**_attrs(op), "scale": scale})
    if op == "CACHE_READ":
        with pytest.raises(ValueError, match="length"):
            check_op(op, shapes, dtypes, LAY.attrs)
    if op != "VERIFY_DRAFT":
        with pytest.raises(ValueError, match="page_size"):
            check_op(op, shapes, dtypes, {**_attrs(op), "page_size": 24})


def test_plan_keeps_the_state_out_of_the_arena():
    g = step_graph(read=6)
    assert not [r for r in run_validators(Phase.POST_OPTIMIZE, g)]
    mem = plan(g)
    assert "cache" not in mem.offsets and "cache2" not in mem.offsets
    assert [n.op for n in mem.order][0] == OpType.CACHE_WRITE
    check_extents(dispatch_order(mem), g)
    assert g.state_of("cache2") == "cache" and g.state_of("q") is None


def test_a_write_alone_is_not_dead():
    g = step_graph()
    g.outputs = []
    g.remove_node([n.id for n in g if n.op == OpType.PAGED_ATTENTION][0])
    run_pipeline(g)
    assert [n.op for n in g] == [OpType.CACHE_WRITE] and g.states == ["cache"]


def test_reader_of_the_value_before_a_write_is_an_error():
    g = step_graph()
    _tensor(g, "z", (2, 3, 2, 6, 24), role="outputs")
    g.add_node(OpType.CACHE_READ, ["cache", "table", "start", "count"], "z", {**LAY.attrs, "length": 6})
    with pytest.raises(Exception, match="let it use 'cache2'"):
        run_validators(Phase.POST_OPTIMIZE, g)


def test_writing_an_input_is_an_error():
    g = step_graph()
    g.states, g.inputs = [], g.inputs + ["cache"]
    with pytest.raises(Exception, match="not a state"):
        run_validators(Phase.POST_OPTIMIZE, g)
    with pytest.raises(ValueError, match="not a state"):
        check_extents(list(g), g)


def test_graph_file_keeps_states(tmp_path):
    g = step_graph()
    g.save(tmp_path / "g")
    h = Graph.load(tmp_path / "g")
    assert h.states == ["cache"] and h.to_dict() == g.to_dict()
    assert "states" not in Graph().to_dict()


def test_library_takes_the_nodes():
    lib = open_library()
    g = step_graph(read=6)
    arr, order = host_nodes(g)
    assert lib.check_nodes(arr, len(order), []) == len(order) == 3


FIELDS = [("extra", 0, [0, 8, 24, 65536, -16]), ("extra", 1, [0, -1, 1 << 30]), ("extra", 2, [0, 257, -1]),
          ("extra", 3, [-1, 4]), ("extra", 4, [0, -3]), ("extra", 5, [0, -1, 1 << 30]), ("n_dims", None, [1, 3, 6]),
          ("n_inputs", None, [0, 2, 12]), ("elem_size", None, [2])]


@pytest.mark.parametrize("at", [0, 1, 2])
def test_library_refuses_malformed_cache_nodes(at):
    lib = open_library()
    g = step_graph(read=6)
    for field, k, values in FIELDS:
        for v in values:
            arr, order = host_nodes(g)
            if k is None:
                setattr(arr[at], field, v)
            else:
                getattr(arr[at], field)[k] = v
            with pytest.raises(HipExecutorError):
                lib.check_nodes(arr, len(order), [])
    for j in range(arr[at].n_inputs):
        arr, order = host_nodes(g)
        arr[at].inputs[j] = None
        with pytest.raises(HipExecutorError, match="null"):
            lib.check_nodes(arr, len(order), [])
    arr, order = host_nodes(g)
    cache = 1 if order[at].op == OpType.PAGED_ATTENTION else 0
    arr[at].inputs[cache] += 4
    with pytest.raises(HipExecutorError):
        lib.check_nodes(arr, len(order), [])


def verify_node(B=2, D=3, V=50):
    n = COpNode()
    n.op, n.n_inputs, n.n_dims, n.elem_size = OpType.VERIFY_DRAFT.value, 5, 2, 8
    for k in range(5):
        n.inputs[k] = (k + 1) << 20
    n.output = 1 << 24
    n.out_shape[0], n.out_shape[1], n.extra[0] = B, D + 1, V
    return (COpNode * 1)(n)


def test_library_refuses_malformed_verify_nodes():
    lib = open_library()
    assert lib.check_nodes(verify_node(), 1, []) == 1
    assert lib.check_nodes(verify_node(D=0), 1, []) == 1
    for bad in (verify_node(B=65536), verify_node(D=-1), verify_node(V=0), verify_node(V=(1 << 30) + 1)):
        with pytest.raises(HipExecutorError):
            lib.check_nodes(bad, 1, [])
    for k in range(5):
        n = verify_node()
        n[0].inputs[k] = None
        with pytest.raises(HipExecutorError):
            lib.check_nodes(n, 1, [])
        n = verify_node()
        n[0].inputs[k] += 2
        with pytest.raises(HipExecutorError):
            lib.check_nodes(n, 1, [])


def test_library_survives_random_fields():
    """Records with a few random fields: steps or an error, under the sanitizers too."""
    lib = open_library()
    r = np.random.default_rng(3)
    ints = [-(1 << 31), -7, -1, 0, 1, 2, 3, 4, 5, 16, 64, 256, 1000, 65535, 1 << 20, (1 << 31) - 1]
    base = []
    for g in (step_graph(read=6), step_graph(CacheLayout(1, 128, 64, "float32"), 1, 8, 1, 2, 2)):
        base.append(host_nodes(g))
    for trial in range(400):
        src, order = base[trial % 2] if trial % 3 else (verify_node(), [None])
        n = len(order)
        arr = (COpNode * n)()
        ctypes.memmove(arr, src, ctypes.sizeof(COpNode) * n)
        for _ in range(int(r.integers(1, 4))):
            nd = arr[int(r.integers(n))]
            v = ints[int(r.integers(len(ints)))]
            k = int(r.integers(5))
            if k == 0:
                nd.extra[int(r.integers(8))] = v
            elif k == 1:
                nd.out_shape[int(r.integers(5))] = v
            elif k == 2:
                nd.n_dims = int(r.integers(0, 7))
            elif k == 3:
                nd.n_inputs = int(r.integers(0, 13))
            else:
                nd.op = int(r.integers(1100, 1104))
        for fuse in (False, True):
            try:
                assert 0 <= lib.check_nodes(arr, n, [(1 << 20, 4096)], fuse=fuse) <= n
            except HipExecutorError:
                pass


# ---------------------------------------------------------------- the reference itself

def test_reference_types_against_torch():
    torch = pytest.importorskip("torch")
    t = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(t, e4m3_table())
    x = np.random.default_rng(0).standard_normal(4000).astype(np.float32)
    x[0] = 448.0                    # scale 1: the stored values are e4m3's roundings of x
    y, s = store(x, "float8")
    assert s == 1.0
    np.testing.assert_array_equal(y, torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy())


def test_reference_scales():
    for kind in CACHE_TYPES:
        assert row_scale(np.zeros(4, np.float32), kind) == 2.0**-126
        assert np.isnan(row_scale(np.array([1, np.inf], np.float32), kind))
        row = np.array([3.0, -2.5e-3, 1e-7], np.float32)
        y, s = store(row, kind)
        step = {"float32": 0, "float16": 2.0**-12 * 3, "int8": s / 2, "float8": s * 16}[kind]
        assert np.abs(y * s - row).max() <= step
    assert row_scale(np.array([3.0]), "float16") == 2.0**-13


def test_reference_pack_is_the_layout():
    """Byte addresses of single elements, from the layout's words."""
    lay = CacheLayout(2, 20, 32, "float16")
    p = Pages.random(lay, 2, np.random.default_rng(1))
    raw = p.pack()
    for page, h, slot, d in ((0, 0, 0, 0), (1, 1, 31, 19), (1, 0, 13, 7)):
        head = raw[page, h * lay.head_bytes:(h + 1) * lay.head_bytes]
        k = head[:32 * 32 * 2].view(np.float16)
        v = head[32 * 32 * 2:2 * 32 * 32 * 2].view(np.float16)
        s = head[2 * 32 * 32 * 2:].view(np.float32)
        assert k[slot * 32 + d] == p.y[page, h, 0, slot, d]
        assert v[(slot // 8 * 32 + d) * 8 + slot % 8] == p.y[page, h, 1, slot, d]
        assert s[slot] == p.s[page, h, 0, slot] and s[32 + slot] == p.s[page, h, 1, slot]


@pytest.mark.parametrize("read", [1, 5, 6, 40])
def test_plan_keeps_every_output(read):
    """An output that no later node takes stays where it is until the end, whatever is computed behind it."""
    g = step_graph(batch=1, heads=2, chunk=read, read=read)
    mem = plan(g)
    assert not run_validators(Phase.POST_PLAN, mem)
    span = {n: (mem.offsets[n], mem.offsets[n] + 4 * int(np.prod(g.tensors[n].shape))) for n in g.outputs}
    (a0, a1), (b0, b1) = span.values()
    assert a1 <= b0 or b1 <= a0


def test_plan_overwrites_no_output_in_place():
    g = Graph()
    _tensor(g, "x", (8, 8))
    _tensor(g, "y", (8, 8), role="outputs")
    _tensor(g, "z", (8, 8), role="outputs")
    g.add_node(OpType.EXP, ["x"], "y")
    g.add_node(OpType.RELU, ["y"], "z")
    mem = plan(g)
    assert not run_validators(Phase.POST_PLAN, mem)
    assert mem.offsets["y"] != mem.offsets["z"]


def test_graph_file_keeps_what_a_state_holds_at_first(tmp_path):
    g = step_graph()
    r = np.random.default_rng(0)
    g.tensors["cache"].buffer = r.integers(0, 256, g.tensors["cache"].shape, dtype=np.uint8)
    g.save(tmp_path / "g")
    np.testing.assert_array_equal(Graph.load(tmp_path / "g").tensors["cache"].buffer, g.tensors["cache"].buffer)


class OnDevice:
    """What a tensor in device memory shows of itself."""

    def __init__(self, shape=(4, 6), typestr="<f4", at=1 << 20, strides=None, index=0):
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (at, False), "strides": strides,
                                         "version": 2}
        self.device = type("Device", (), {"index": index})()


def test_device_tensors_are_checked_against_the_graph():
    from runtime.executor.compiled import _device_range

    def address(t):
        return _device_range(t, "q", (4, 6), "float32", 0)

    assert address(OnDevice()) == address(OnDevice(strides=(24, 4))) == 1 << 20
    for bad, error in ((np.zeros((4, 6), np.float32), "not in device memory"), (OnDevice(index=1), "on device 1"),
                       (OnDevice(shape=(6, 4)), "shape"), (OnDevice(typestr="<f8"), "float64"),
                       (OnDevice(strides=(4, 16)), "contiguous"), (OnDevice(strides=(48, 4)), "contiguous"),
                       (OnDevice(at=(1 << 20) + 4), "16-byte")):
        with pytest.raises((TypeError, ValueError), match=error):
            address(bad)
