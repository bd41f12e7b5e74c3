"""The operators of residual blocks with experts where a call has next to nothing to do, where operands alias, and where sizes
pass a threshold between kernels; beside tests/test_gpu_blocks.py, whose formulas and bars they use."""
import numpy as np
import pytest

from cortex_amd import blocks
from cortex_amd import capi
from cortex_amd import driver as drv
from cortex_amd import optimize
from cortex_amd import tensor as ct
from test_gpu_blocks import D, Owned, as_released, read, run_route, stream, strides_of  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu


def part(D, whole, at, shape):
    """A dense tensor of `shape` whose elements are those of the vector `whole` from `at` on; perhaps none."""
    return ct.Tensor(whole.device, {"shape": list(shape), "strides": strides_of(shape)}, whole.buffer.sub_buffer(at, int(np.prod(shape))))


# ------------------------------------------------------------------------------------------------- norms of nothing

@pytest.mark.parametrize("biases", [False, True])
@pytest.mark.parametrize("gate", [(0, 50), (0, 1), (1, 50), (1, 1)], ids=str)
def test_norm_gradient_of_no_rows_stays_inside_its_gradients(D, gate, biases):
    """The gradients are parts of one buffer, as those of a network often are: those that have elements are zeros, and what lies
    behind one that has none is not written."""
    width = 50
    shapes = {"post-scale": (width,), "pre-scale": (width,), "gate": gate}
    if biases:
        shapes.update({"post-bias": (width,), "pre-bias": (width,)})
    guard = 64
    total = sum(int(np.prod(s)) + guard for s in shapes.values())
    values, flat, want = D.tensor(np.ones(total)), D.tensor(np.full(total, 7.25)), np.full(total, 7.25)
    p, g, at = {}, {}, 0
    for k, s in shapes.items():
        p[k], g[k] = part(D, values, at, s), part(D, flat, at, s)
        want[at:at + int(np.prod(s))] = 0
        at += int(np.prod(s)) + guard
    empty = [D.tensor(np.zeros((0, width))) for _ in range(4)]
    d = blocks.norm_descriptor(post="layer", pre="rms")
    blocks.norm_residual(empty[0], empty[1], None, empty[2], empty[3], p, d)
    blocks.norm_residual_gradient(empty[0], empty[1], g, empty[2], empty[3], empty[0], empty[1], None, p, d)
    assert np.array_equal(read(flat), want)


@pytest.mark.parametrize("gate", [(7, 1), (1, 1), (7, 0), (1, 0)], ids=str)
def test_norm_gradient_of_rows_without_elements(D, gate):
    """A gate's gradient that has elements is a sum of nothing: zeros, and no more of them than it has."""
    rows, n = 7, int(np.prod(gate))
    flat, empty = D.tensor(np.full(20, 7.25)), [D.tensor(np.zeros((rows, 0))) for _ in range(4)]
    p, g = {"gate": part(D, D.tensor(np.ones(20)), 0, gate)}, {"gate": part(D, flat, 2, gate)}
    d = blocks.norm_descriptor(post="rms", pre="none")
    blocks.norm_residual_gradient(empty[0], empty[1], g, empty[2], None, empty[3], empty[3], D.tensor(np.zeros((4, rows))), p, d)
    want = np.full(20, 7.25)
    want[2:2 + n] = 0
    assert np.array_equal(read(flat), want)


def test_norm_gradients_between_the_rows_of_an_operand(D):
    """Vectors in the columns that a wider matrix has beside the operand overlap nothing of it, and are taken."""
    rng = np.random.default_rng(62)
    rows, width, wide = 5, 24, 100
    whole = D.tensor(rng.standard_normal(rows * wide))
    z = ct.Tensor(whole.device, {"shape": [rows, width], "strides": [wide, 1]}, whole.buffer)
    p = {k: D.tensor(rng.standard_normal(width)) for k in ("post-scale", "post-bias", "pre-scale")}
    d = blocks.norm_descriptor(post="layer", pre="rms")
    out, h, stats, dout, dh = (D.tensor(rng.standard_normal(s)) for s in ([(rows, width)] * 2 + [(4, rows)] + [(rows, width)] * 2))
    blocks.norm_residual(out, h, stats, z, None, p, d)
    results = []
    for between in (False, True):
        g = {k: part(D, whole, wide * i + width + 3 * i, (width,)) if between else D.tensor(np.zeros(width)) for i, k in enumerate(p)}
        dz = D.tensor(np.zeros((rows, width)))
        blocks.norm_residual_gradient(dz, None, g, dout, dh, z, out, stats, p, d)
        results.append([read(dz)] + [read(t) for t in g.values()])
    for a, b in zip(*results):
        assert np.array_equal(a, b) and np.any(a != 0)


def test_norm_gradient_of_a_row_of_more_columns_than_a_launch_s_lanes(stream):
    """The columns' sums of a row of over 2^27 floats.  All ones by a scale of ones and an epsilon of 3: the rate is exactly a half, the
    sum over the row of y zh is its length over 2, and the row's gradient (1 - 1 / 4) / 2."""
    D = Owned("float")
    width = (1 << 27) + 33
    ones = np.ones((1, width), np.float32)
    d = blocks.norm_descriptor(post="rms", pre="none", epsilon=3.0)
    z, out, scale, dz, dr = (D.tensor(x) for x in (ones, ones, ones[0], 0 * ones, 0 * ones))
    stats, g = D.tensor(np.zeros((4, 1))), {"post-scale": D.tensor(np.full(width, 3.0, np.float32))}
    blocks.norm_residual(out, None, stats, z, None, {"post-scale": scale}, d)
    assert np.array_equal(read(stats)[:, 0], [0, 0.5, 0, 1]) and np.all(read(out) == 0.5)
    blocks.norm_residual_gradient(dz, dr, g, z, None, z, out, stats, {"post-scale": scale}, d)
    assert np.all(read(g["post-scale"]) == 0.5) and np.all(read(dz) == 0.375) and np.all(read(dr) == 1)
    D.free()


@pytest.mark.parametrize("shape", [(6, 3), (37, 70), (300, 300), (9, 5003), (2, 17000)], ids=str)
@pytest.mark.parametrize("by_column", [False, True])
def test_norms_with_a_gate_whose_rows_lie_apart(D, shape, by_column):
    """A full gate, or one of a value to a row, that is a block of a wider matrix: the same bits as of one by itself."""
    rows, width = shape
    rng = np.random.default_rng(68)
    gate = rng.standard_normal((rows, width if by_column else 1))
    z, dout, dh = (D.tensor(rng.standard_normal((rows, width))) for _ in range(3))
    p = {"post-scale": D.tensor(rng.standard_normal(width)), "post-bias": D.tensor(rng.standard_normal(width))}
    d = blocks.norm_descriptor(post="rms", pre="layer")
    results = []
    for given in (D.tensor(gate), D.block(gate, 5)):
        q = {**p, "gate": given}
        out, h, dz, dr = (D.tensor(np.zeros((rows, width))) for _ in range(4))
        stats, g = D.tensor(np.zeros((4, rows))), {k: D.tensor(np.full(t.shape(), 3.0)) for k, t in q.items()}
        blocks.norm_residual(out, h, stats, z, None, q, d)
        blocks.norm_residual_gradient(dz, dr, g, dout, dh, z, out, stats, q, d)
        results.append([read(t) for t in (out, h, stats, dz, dr, *g.values())])
    for a, b in zip(*results):
        assert np.array_equal(a, b) and np.any(a != 0)


# ------------------------------------------------------------------------------------------------- routing

@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("size", [(1, 3, 2), (50, 7, 3), (40, 30, 2), (33, 61, 8), (21, 130, 4), (9, 1021, 5), (3000, 257, 2)], ids=str)
def test_route_gradient_in_place_of_the_logits(D, size, renormalize):
    """The same bits as into memory of its own, rows apart and with widths that end inside a piece."""
    n, e, k = size
    rng = np.random.default_rng(63)
    logits = rng.standard_normal((n, e))
    logits[rng.random((n, e)) < 0.2] = -np.inf
    apart, to = D.block(logits, 3), D.block(np.zeros((n, e)), 3)
    t, (experts, weights, *_) = run_route(D, logits, k, renormalize)
    dw = D.tensor(rng.standard_normal((n, k)))
    blocks.route_experts_gradient(to, dw, weights, experts, apart, renormalize=renormalize)
    blocks.route_experts_gradient(apart, dw, weights, experts, apart, renormalize=renormalize)
    assert np.array_equal(read(apart), read(to)) and np.any(read(to) != 0)


def test_routing_is_recorded_with_the_scratch_that_it_is_said_to_need(as_released):
    """8 MiB reserved ahead: the most counts that there are, and their totals, fit; nothing is allocated while the stream is captured."""
    import ctypes as C
    rt = C.CDLL("libamdhip64.so")
    rt.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    rt.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    rt.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    rt.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    rt.hipGraphExecDestroy.argtypes = rt.hipGraphDestroy.argtypes = [C.c_void_p]
    device = drv.HipDriver().default_device()
    stream, loader = device.create_stream(), device.create_stream()
    capi.call("ct_stream_reserve_scratch", stream.handle, 8 << 20, 0)
    n, e = 64 * 2048, 1023
    D = Owned("float")
    with ct.tensor_context(loader, "float"):
        logits = ct.new_tensor([n, e])
        D.kept.append(logits)
        results = [D.tensor(np.full(s, 77), kind) for s, kind in (((n, 1), "int"), ((n, 1), "float"), ((e + 1,), "int"), ((n,), "int"), ((n, 1), "int"))]
        blocks.route_experts(*results, logits)     # the kernels are loaded
        want = [read(t) for t in results]
        assert np.all(want[0] == 0) and np.all(want[1] == 1) and want[2].tolist() == [0] + [n] * e and np.array_equal(want[3], np.arange(n))
        for t in results:
            capi.call("ct_memset", loader.handle, t.buffer.ptr, capi.DTYPE_CODES[t.get_datatype()], 77.0, t.ecount())
        capi.call("ct_stream_sync", loader.handle)
    with ct.tensor_context(stream, "float"):
        graph, graph_exec = C.c_void_p(), C.c_void_p()
        assert rt.hipStreamBeginCapture(stream.handle, 1) == 0
        try:
            blocks.route_experts(*results, logits)
        finally:
            ended = rt.hipStreamEndCapture(stream.handle, C.byref(graph))
        assert ended == 0 and graph.value
        assert rt.hipGraphInstantiate(C.byref(graph_exec), graph, None, None, 0) == 0
        for _ in range(2):
            assert rt.hipGraphLaunch(graph_exec, stream.handle) == 0
            for a, b in zip(want, results):
                assert np.array_equal(a, read(b))
        capi.call("ct_stream_sync", stream.handle)
        assert rt.hipGraphExecDestroy(graph_exec) == 0 and rt.hipGraphDestroy(graph) == 0
        D.free()
    stream.release()
    loader.release()


# ------------------------------------------------------------------------------------------------- products of very many tiles

def test_products_of_more_tiles_than_a_launch_takes(D, stream):
    """Over 2^21 tiles of 16 rows (32 of doubles), k below a tile's and a single column.  Whole numbers: every sum exact."""
    rng = np.random.default_rng(65)
    rows, k = ((1 << 25) + 37, 2) if D.datatype == "float" else ((1 << 26) + 100, 1)
    cuts = [5, 5 + (1 << 20), rows - 3]
    a, b = rng.integers(-7, 8, (rows, k), np.int8).astype(D.type), rng.integers(1, 8, (3, 1, k)).astype(D.type)
    c = D.tensor(np.full((rows, 1), 7.25))
    blocks.grouped_gemm(c, True, 1.0, D.tensor(a), D.tensor(b), 0.0, D.tensor([cuts[0], cuts[1], cuts[1], cuts[2]], "int"))
    got = read(c)
    assert np.all(got[:cuts[0]] == 7.25) and np.all(got[cuts[2]:] == 7.25)
    for e, i in ((0, slice(cuts[0], cuts[1])), (2, slice(cuts[1], cuts[2]))):
        assert np.array_equal(got[i, 0], a[i] @ b[e, 0])


def test_products_over_rows_of_more_tiles_than_a_launch_takes(D):
    """65535 groups of 33 tiles, most of them without rows: the products of those that have some, zeros in all others."""
    rng = np.random.default_rng(66)
    groups, rows, n = 65535, 300, 2049 if D.datatype == "float" else 1025
    group_of = np.sort(rng.integers(0, groups, rows))
    group_of[-1] = groups - 1
    offsets = np.searchsorted(group_of, np.arange(groups + 1))
    a, b = rng.integers(-7, 8, (rows, 1)).astype(D.type), rng.integers(-7, 8, (rows, n)).astype(D.type)
    c = D.tensor(np.full((groups, 1, n), 7.25))
    blocks.grouped_gemm_weights(c, 1.0, D.tensor(a), D.tensor(b), 0.0, D.tensor(offsets, "int"))
    want = np.zeros((groups, n), D.type)
    np.add.at(want, group_of, a * b)
    assert np.array_equal(read(c)[:, 0], want)


def test_products_without_terms_over_very_many_rows(D, stream):
    """More row tiles than a launch has rows of blocks: beta times what was there, in the groups' rows."""
    rows, n, code = 5_000_000, 3, capi.DTYPE_CODES[D.datatype]
    c = np.arange(rows * n, dtype=np.int64).reshape(rows, n) % 1021 + 1.0
    offsets, tc = D.tensor([7, 4_500_000, rows - 9], "int"), D.tensor(c)
    capi.call("ct_grouped_gemm", stream.handle, tc.buffer.ptr, n, 1, 1.0, None, rows, 0, 4, None, None, n, 4, 0, offsets.buffer.ptr, 2, rows, 0.5, code)
    c[7:rows - 9] *= 0.5
    assert np.array_equal(read(tc), c.astype(D.type))


def test_products_over_rows_far_apart_of_very_many_columns(stream):
    D = Owned("float")
    rng = np.random.default_rng(67)
    m, ld = 65535 * 64 + 100, (1 << 30) + 5
    x, y = rng.integers(-7, 8, (2, m)).astype(np.float32), np.array([[2], [-3]], np.float32)
    far = ct.new_tensor([ld + m], datatype="float")
    D.kept.append(far)
    for r in range(2):
        row = D.tensor(x[r])
        capi.call("ct_memcpy_async", far.buffer.ptr + 4 * ld * r, row.buffer.ptr, 4 * m, capi.COPY_D2D, stream.handle)
    w = D.tensor(np.zeros((1, m, 1)))
    capi.call("ct_grouped_gemm_weights", stream.handle, w.buffer.ptr, 1, m, 1.0, far.buffer.ptr, 2, m, ld, None, D.tensor(y).buffer.ptr, 2, 1, 1, None,
              D.tensor([0, 2], "int").buffer.ptr, 1, 2, 0.0, capi.F32)
    assert np.array_equal(read(w)[0], x.T @ y)
    D.free()


# ------------------------------------------------------------------------------------------------- combining

@pytest.mark.parametrize("size", [(1, 1, 1), (40, 3, 33), (700, 2, 1000), (3, 4, 4100), (300, 4, 2050)], ids=str)
def test_combine_gradient_in_place_of_the_weights(D, size):
    """The same bits as into memory of its own, with 16, 64 and 256 lanes to an assignment."""
    n, k, width = size
    rng = np.random.default_rng(64)
    rows, dy = D.tensor(rng.standard_normal((n * k, width))), D.tensor(rng.standard_normal((n, width)))
    slots, weights = D.tensor(rng.permutation(n * k).reshape(n, k), "int"), D.tensor(rng.standard_normal((n, k)))
    to = [D.tensor(np.zeros((n * k, width))) for _ in range(2)]
    apart = D.tensor(np.zeros((n, k)))
    blocks.combine_experts_gradient(to[0], apart, dy, rows, weights, slots)
    blocks.combine_experts_gradient(to[1], weights, dy, rows, weights, slots)
    assert np.array_equal(read(weights), read(apart)) and np.array_equal(read(to[0]), read(to[1])) and np.any(read(apart) != 0)


# ------------------------------------------------------------------------------------------------- clipping

@pytest.mark.parametrize("n", [2, 50, 120, 121, 300])
def test_clip_gradients_of_tensors_that_touch_in_any_order(D, stream, n):
    """Gradients and outputs side by side in one buffer, shuffled, some in place: nothing overlaps, and each goes where it belongs."""
    rng = np.random.default_rng(n)
    counts = rng.integers(0, 40, n)
    counts[0] = 7
    order = rng.permutation(2 * n)
    ends = np.cumsum(counts[order % n])
    places = np.empty(2 * n, np.int64)
    places[order] = ends - counts[order % n]
    host = rng.standard_normal(int(ends[-1])).astype(D.type)
    flat, result = D.tensor(host), D.tensor(np.zeros(2))
    piece = lambda slot: flat.buffer.sub_buffer(int(places[slot]), int(counts[slot % n]))
    into = [i if rng.random() < 0.5 else n + i for i in range(n)]
    optimize.clip_gradients(optimize.Backend(stream, D.datatype), [piece(i) for i in range(n)], 0.5, result, [piece(i) for i in into])
    norm, factor = read(result)
    values = [host[places[i]:places[i] + counts[i]] for i in range(n)]
    want64 = np.sqrt(sum((v.astype(np.float64) ** 2).sum() for v in values))
    assert abs(float(norm) - want64) <= (4 * D.u + host.size * 2.0 ** -53) * want64
    want = host.copy()
    for i, slot in enumerate(into):
        want[places[slot]:places[slot] + counts[i]] = values[i] * factor
    assert np.array_equal(read(flat), want)


# ------------------------------------------------------------------------------------------------- the layer

@pytest.mark.parametrize("held", [("router",), ("first",), ("second",), ("gate", "post-scale"), ("router", "first", "second", "pre-scale")], ids="-".join)
def test_a_block_with_parameters_that_are_held(D, held):
    """Parameters without a gradient, by None or by its absence: all other gradients are the same bits as with it."""
    rng = np.random.default_rng(61)
    tokens, width, hidden, experts, chosen = 20, 24, 36, 5, 2
    shapes = {"router": (experts, width), "first": (experts, hidden, width), "second": (experts, width, hidden), "post-scale": (width,),
              "pre-scale": (width,), "gate": (1, width)}
    values = {k: D.tensor(rng.standard_normal(s)) for k, s in shapes.items()}
    make = lambda: D.tensor(rng.standard_normal((tokens, width)))
    x, residual, to_output, to_normalized = (make() for _ in range(4))
    results = []
    for how in ("all", "none", "absent"):
        p = {k: {"buffer": v, "gradient": D.tensor(np.full(shapes[k], 3.0))} for k, v in values.items()}
        for k in held if how != "all" else ():
            if how == "none":
                p[k]["gradient"] = None
            else:
                del p[k]["gradient"]
        block = blocks.ExpertBlock(tokens, width, hidden, experts, chosen, datatype=D.datatype)
        output, normalized, dx, dr = (D.tensor(np.zeros((tokens, width))) for _ in range(4))
        block.forward(p, x, residual, output, normalized)
        block.backward(p, x, output, dx, dr, to_output, to_normalized)
        results.append([read(dx), read(dr)] + [read(p[k]["gradient"]) for k in shapes if k not in held])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert np.array_equal(a, b) and np.any(a != 0)
