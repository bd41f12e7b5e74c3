"""The gated product and what its backward pass begins with against their formulas in 64 bits (numpy), the blocks that are made of
them against differences.

Bars, fixed ahead, with u = 2^-24 (float) or 2^-53 (double): a sum of k products taken one after the other is held to (k + 4) u of the sum
of its terms' magnitudes.  The results carry that on: no activation here is steeper than 1.2, and an activation and its derivative
are each evaluated in a few roundings of terms that are below 1.5 (times the argument, where it is a factor), which 32 u of those
terms cover.
"""
import ctypes as C
import math

import numpy as np
import pytest

from cortex_amd import blocks
from cortex_amd import capi
from cortex_amd import driver as drv
from cortex_amd import optimize
from cortex_amd import tensor as ct
from test_gpu_blocks import NUMPY, UNIT, Owned, as_released, close, read, stream  # noqa: F401

pytestmark = pytest.mark.gpu

_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def activation64(kind, g):
    """f, f', and the magnitudes of what they are formed of."""
    with np.errstate(over="ignore"):
        p = 1 / (1 + np.exp(-g))
        rest = 1 / (1 + np.exp(g))
    if kind == "swish":
        return g * p, p + g * p * rest, abs(g) * p, p + abs(g) * p * rest
    if kind == "logistic":
        return p, p * rest, p, p * rest
    if kind == "tanh":
        t = np.tanh(g)
        return t, 1 / np.cosh(np.minimum(abs(g), 300)) ** 2, abs(t), np.ones_like(g)     # 1 - t is rounded where t is near 1
    if kind == "gelu":
        share, bell = 0.5 * _erfc(-g / math.sqrt(2)), np.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        # an argument's rounding moves the exponential by x^2 as many parts
        return g * share, share + g * bell, (1 + g * g) * abs(g) * share, share + (1 + g * g) * abs(g) * bell + (1 + g * g) * share
    return np.maximum(g, 0), (g > 0).astype(np.float64), np.maximum(g, 0), (g > 0).astype(np.float64)


@pytest.fixture(params=["float", "double"])
def D(request, stream):  # noqa: F811
    owned = Owned(request.param)
    owned.u, owned.type = UNIT[request.param], NUMPY[request.param]
    yield owned
    owned.free()


def groups_of(rng, rows, groups, kind):
    """Offsets of groups of uneven sizes, some of none; rows before the first and behind the last group."""
    if groups is None:
        return None, [(0, rows)]
    first, last = (rows // 10, rows - rows // 8) if kind == "gaps" else (0, rows)
    cuts = np.sort(rng.integers(first, last + 1, groups - 1))
    offsets = np.concatenate([[first], cuts, [last]])
    return offsets, list(zip(offsets[:-1], offsets[1:]))


def check(D, rows, width, hidden, groups=None, activation="swish", kind="", indexed=False, keep=True, pad=0, seed=0):
    rng = np.random.default_rng(seed)
    a_rows = rows + 7 if indexed else rows
    offsets, ranges = groups_of(rng, rows, groups, kind)
    n_groups = 1 if groups is None else groups
    x = rng.standard_normal((a_rows, width))
    first = rng.standard_normal((n_groups, 2 * hidden, width)) * 1.5 / math.sqrt(max(width, 1))
    second = rng.standard_normal((n_groups, width, hidden)) / math.sqrt(hidden)
    dy = rng.standard_normal((rows, width))
    index = rng.integers(-1, a_rows + 2, rows) if indexed else None
    place = (lambda v: D.block(v, pad)) if pad else D.tensor
    tx, tdy = place(x), place(dy)
    tfirst, tsecond = (D.tensor(first), D.tensor(second)) if groups else (place(first[0]), place(second[0]))
    inner, pre, pre_gradient, again = (place(np.full((rows, n), 3.5)) for n in (hidden, 2 * hidden, 2 * hidden, hidden))
    toffsets = None if groups is None else D.tensor(offsets, "int")
    tindex = None if index is None else D.tensor(index, "int")
    blocks.gated_gemm(inner, pre if keep else None, tx, tfirst, toffsets, tindex, activation=activation)
    met = [capi.last_kernel()]
    x, first, second, dy = (read(t).astype(np.float64) for t in (tx, tfirst, tsecond, tdy))
    first, second = first.reshape(n_groups, 2 * hidden, width), second.reshape(n_groups, width, hidden)
    got, got_pre = read(inner).astype(np.float64), read(pre).astype(np.float64)
    if not keep:
        assert np.all(got_pre == 3.5)
        pre.buffer and ct.assign(pre, 0.0)
    inside = np.zeros(rows, bool)
    for g, (a, b) in enumerate(ranges):
        inside[a:b] = True
        taken = x[a:b] if index is None else np.where(((index[a:b] >= 0) & (index[a:b] < a_rows))[:, None], x[np.clip(index[a:b], 0, a_rows - 1)], 0)
        want, scale = taken @ first[g].T, (width + 4) * D.u * (abs(taken) @ abs(first[g]).T)
        if keep:
            close(got_pre[a:b], want, scale, 1.0, "pre")
        gate, up = want[:, :hidden], want[:, hidden:]
        f, _, f_scale, _ = activation64(activation, gate)
        bar = 1.2 * scale[:, :hidden] * (abs(up) + scale[:, hidden:]) + (abs(f) + 1e-30) * scale[:, hidden:] + 32 * D.u * f_scale * abs(up)
        close(got[a:b], f * up, bar + 1e-38, 1.0, "inner")
    assert np.all(got[~inside] == 3.5) and (not keep or np.all(got_pre[~inside] == 3.5))
    if keep:
        blocks.gated_gemm_gradient(pre_gradient, again if seed % 2 else None, tdy, tsecond, pre, toffsets, activation=activation)
        met.append(capi.last_kernel())
        result, back = read(pre_gradient).astype(np.float64), read(again).astype(np.float64)
        for g, (a, b) in enumerate(ranges):
            d, scale = dy[a:b] @ second[g], (width + 4) * D.u * (abs(dy[a:b]) @ abs(second[g]))
            gate, up = got_pre[a:b, :hidden], got_pre[a:b, hidden:]
            f, slope, f_scale, slope_scale = activation64(activation, gate)
            close(result[a:b, :hidden], d * up * slope, abs(up) * (scale * abs(slope) + 32 * D.u * abs(d) * slope_scale) + 1e-38, 1.0, "gate's gradient")
            close(result[a:b, hidden:], d * f, scale * abs(f) + 32 * D.u * abs(d) * f_scale + 1e-38, 1.0, "up's gradient")
            if seed % 2:
                assert np.array_equal(back[a:b], got[a:b]), "the inner rows once more"
        assert np.all(result[~inside] == 3.5) and np.all(back[~inside if seed % 2 else slice(None)] == 3.5)
        blocks.gated_gemm_gradient(pre, None, tdy, tsecond, pre, toffsets, activation=activation)     # in place
        assert np.array_equal(read(pre), result.astype(D.type))
    return met


SIZES = [(1, 1, 1), (1, 7, 3), (3, 31, 5), (5, 33, 17), (16, 64, 40), (17, 100, 33), (40, 257, 65), (130, 96, 64), (1, 2048, 300), (70, 1111, 129)]


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_dense(D, size):
    check(D, *size, seed=1)


@pytest.mark.parametrize("activation", blocks.GATES)
def test_activations(D, activation):
    for seed in (0, 1):
        check(D, 40, 70, 50, activation=activation, seed=seed)
        check(D, 90, 40, 33, 4, activation=activation, seed=seed)


@pytest.mark.parametrize("indexed", [False, True])
@pytest.mark.parametrize("kind", ["", "gaps"])
def test_groups(D, kind, indexed):
    check(D, 200, 64, 48, 5, kind=kind, indexed=indexed)
    check(D, 33, 50, 7, 70, kind=kind, indexed=indexed, activation="gelu", seed=1)     # more groups than rows
    check(D, 1500, 130, 100, 3, kind=kind, indexed=indexed, seed=2)


def test_rows_apart(D):
    check(D, 60, 50, 35, pad=3, seed=1)
    check(D, 300, 70, 129, pad=1, keep=False)
    check(D, 20, 31, 9, 3, pad=2, indexed=True)


def test_each_kernel_of_floats(stream):  # noqa: F811
    """Sizes that between them meet every kernel, whatever the choice among them is measured to be at one of them."""
    D, met = Owned("float"), set()
    D.u, D.type = UNIT["float"], np.float32
    for size in ((16, 640, 5000), (3, 1024, 200), (600, 256, 640), (4096, 160, 1030), (128, 4096, 96), (2048, 2048, 64), (40, 1000, 130), (2, 20, 40),
                 (700, 64, 1100), (200, 4096, 130), (512, 2048, 64), (100, 8192, 300), (3000, 1000, 2300), (2048, 512, 1024, 8), (2048, 512, 2048, 8)):
        met.update(check(D, *size, seed=1))
        D.free()
        D.kept.clear()
    assert met >= {"gated_thin", "gated_gradient_thin", "gated_medium", "gated_gradient_medium", "gated_large", "gated_gradient_large",
                   "gated_medium+gated_sum", "gated_gradient_medium+gated_sum", "gated_pairs", "gated_gradient_pairs"}, met


def test_many_rows_of_floats_by_group(stream):  # noqa: F811
    """Groups of uneven sizes, rows by index and rows of no group, with two halves to a float."""
    D = Owned("float")
    D.u, D.type = UNIT["float"], np.float32
    for kwargs in ({}, {"indexed": True, "kind": "gaps"}, {"pad": 3, "activation": "gelu"}):
        assert check(D, 5000, 1000, 2300, 3, seed=1, **kwargs) == ["gated_pairs", "gated_gradient_pairs"]
        D.free()
        D.kept.clear()


def test_rows_of_any_magnitude(stream):  # noqa: F811
    """With two halves to a float each row and column has its power of two: magnitudes from the smallest to the largest ones, rows of zeros,
    and elements far below the largest of their row, whose products are held to the float sum's bar."""
    D = Owned("float")
    rng = np.random.default_rng(7)
    rows, width, hidden = 3000, 1000, 2300
    x = rng.standard_normal((rows, width)).astype(np.float32)
    weights = (rng.standard_normal((2 * hidden, width)) / math.sqrt(width)).astype(np.float32)
    x *= np.exp2(rng.integers(-60, 30, rows)).astype(np.float32)[:, None]
    x[5], x[6, 1:], x[7] = 0, 0, np.float32(1e-42)
    x[:, 17] *= np.float32(2.0 ** 12)            # one channel far above the others, whose weights are small
    weights[:, 17] *= np.float32(2.0 ** -12)
    weights *= np.exp2(rng.integers(-30, 30, 2 * hidden)).astype(np.float32)[:, None]
    inner, pre = D.tensor(np.zeros((rows, hidden))), D.tensor(np.zeros((rows, 2 * hidden)))
    blocks.gated_gemm(inner, pre, D.tensor(x), D.tensor(weights), activation="relu")
    assert capi.last_kernel() == "gated_pairs"
    x, weights = x.astype(np.float64), weights.astype(np.float64)
    close(read(pre), x @ weights.T, (width + 4) * UNIT["float"] * (abs(x) @ abs(weights).T) + 2.0 ** -149, 1.0)
    d = (rng.standard_normal((rows, 1000)) * np.exp2(rng.integers(-40, 40, rows))[:, None]).astype(np.float32)
    back = (rng.standard_normal((1000, hidden)) * np.exp2(rng.integers(-40, 40, hidden))[None]).astype(np.float32)
    ones = D.tensor(np.ones((rows, 2 * hidden)))
    blocks.gated_gemm_gradient(ones, None, D.tensor(d), D.tensor(back), ones, activation="relu")
    assert capi.last_kernel() == "gated_gradient_pairs"
    d, back = d.astype(np.float64), back.astype(np.float64)
    want, bar = d @ back, (1004 + 32) * UNIT["float"] * (abs(d) @ abs(back)) + 2.0 ** -149
    got = read(ones)
    close(got[:, :hidden], want, bar, 1.0)
    close(got[:, hidden:], want, bar, 1.0)
    D.free()


def test_what_is_not_finite_with_two_halves_to_a_float(stream):  # noqa: F811
    """In rows and columns of both operands; absent rows by all of these."""
    D = Owned("float")
    rng = np.random.default_rng(8)
    rows, width, hidden = 3000, 1000, 2300
    x = rng.standard_normal((rows, width)).astype(np.float32)
    weights = rng.standard_normal((2 * hidden, width)).astype(np.float32)
    x[3, 5], x[300, 7], x[301, 8], x[302, 9] = np.nan, np.inf, -np.inf, np.inf
    x[302, 10] = -np.inf
    weights[20, 3], weights[hidden + 40, 4], weights[50, 7] = np.inf, np.nan, 0.0
    index = np.arange(rows)
    index[[8, 2999]] = -1, rows
    inner, pre = D.tensor(np.zeros((rows, hidden))), D.tensor(np.zeros((rows, 2 * hidden)))
    blocks.gated_gemm(inner, pre, D.tensor(x), D.tensor(weights[None]), D.tensor([0, rows], "int"), D.tensor(index, "int"), activation="relu")
    assert capi.last_kernel() == "gated_pairs"
    taken = x.copy()
    taken[[8, 2999]] = 0
    with np.errstate(invalid="ignore"):
        want = taken.astype(np.float64) @ weights.astype(np.float64).T
    got = read(pre)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    rest = np.where(np.isfinite(taken), taken, 0).astype(np.float64)
    scale = (width + 4) * UNIT["float"] * (abs(rest) @ abs(np.where(np.isfinite(weights), weights, 0)).T.astype(np.float64))
    assert np.all(abs(got - want)[fine] <= scale[fine])
    gate, up = got[:, :hidden], got[:, hidden:]
    with np.errstate(invalid="ignore"):
        assert np.array_equal(read(inner), np.maximum(gate, 0) * up, equal_nan=True)
    d, back = x, rng.standard_normal((width, hidden)).astype(np.float32)
    back[3, 30], back[4, 31] = -np.inf, np.nan
    ones = D.tensor(np.ones((rows, 2 * hidden)))
    blocks.gated_gemm_gradient(ones, None, D.tensor(d), D.tensor(back), ones, activation="relu")
    assert capi.last_kernel() == "gated_gradient_pairs"
    with np.errstate(invalid="ignore"):
        want = d.astype(np.float64) @ back.astype(np.float64)
    got = read(ones)[:, :hidden]
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    D.free()


def test_long_sums_of_doubles(stream):  # noqa: F811
    D, met = Owned("double"), set()
    D.u, D.type = UNIT["double"], np.float64
    for size in ((30, 3000, 20), (700, 40, 600)):
        met.update(check(D, *size, seed=1))
    assert met == {"gated_double", "gated_gradient_double", "gated_double+gated_sum", "gated_gradient_double+gated_sum"}, met
    D.free()


@pytest.mark.parametrize("size", [(2, 256, 146), (2, 352, 33), (33, 400, 64), (1, 464, 7), (17, 300, 128), (40, 255, 96)], ids=str)
def test_sums_of_some_hundred_terms_by_few_rows(D, size):
    """Rows whole lines and parts of lines apart, in products that take every wave several runs of k."""
    check(D, *size, seed=5)
    check(D, *size, activation="gelu", pad=4, seed=6)


def test_sums_of_no_terms(D):
    """Rows without elements, and an operand without rows: gates and ups of zero."""
    for activation in blocks.GATES:
        inner, pre = D.tensor(np.ones((5, 4))), D.tensor(np.ones((5, 8)))
        empty, weights = D.tensor(np.zeros((5, 0))), D.tensor(np.zeros((8, 0)))
        blocks.gated_gemm(inner, pre, empty, weights, activation=activation)
        assert np.all(read(inner) == 0) and np.all(read(pre) == 0)
        blocks.gated_gemm_gradient(pre, inner, empty, D.tensor(np.zeros((0, 4))), pre, activation=activation)
        assert np.all(read(inner) == 0) and np.all(read(pre) == 0)
    inner, index = D.tensor(np.ones((5, 4))), D.tensor(np.arange(5), "int")
    blocks.gated_gemm(inner, None, D.tensor(np.zeros((0, 3))), D.tensor(np.ones((2, 8, 3))), D.tensor([1, 2, 5], "int"), index)
    assert np.array_equal(read(inner), [[1] * 4] + [[0] * 4] * 4)
    none = D.tensor(np.zeros((0, 4)))
    blocks.gated_gemm(none, None, D.tensor(np.zeros((0, 3))), D.tensor(np.ones((8, 3))))
    offsets = D.tensor([0, 0, 0], "int")
    blocks.gated_gemm(inner, None, D.tensor(np.ones((5, 3))), D.tensor(np.ones((2, 8, 3))), offsets)
    assert np.array_equal(read(inner), [[1] * 4] + [[0] * 4] * 4)


def test_offsets_of_any_content(D):
    """Clamped as they are read: no row is written twice or outside."""
    inner = D.tensor(np.full((10, 4), 2.0))
    blocks.gated_gemm(inner, None, D.tensor(np.ones((10, 3))), D.tensor(np.ones((3, 8, 3))), D.tensor([-5, 4, 2, 1 << 30], "int"))
    f = 3 / (1 + math.exp(-3)) * 3
    got = read(inner)
    assert np.all(np.isclose(got[:4], f, rtol=1e-6)) and np.all(np.isclose(got[2:], f, rtol=1e-6))


def test_values_far_out(D):
    """Gates at which exponentials overflow or vanish, and what is not finite: in its own row only."""
    big = 1e4 if D.type == np.float32 else 1e5
    gates = np.array([0.0, -0.0, 1e-30, 20.0, -20.0, 100.0, -100.0, big, -big])
    for activation in blocks.GATES:
        x = np.stack([gates, np.ones_like(gates)], 1)
        weights = np.array([[1.0, 0.0], [0.0, 2.0]])
        inner, pre, tx = D.tensor(np.zeros((9, 1))), D.tensor(np.zeros((9, 2))), D.tensor(x)
        blocks.gated_gemm(inner, pre, tx, D.tensor(weights), activation=activation)
        gate = read(tx)[:, 0].astype(np.float64)
        assert np.array_equal(read(pre)[:, 0], read(tx)[:, 0])
        f, slope, f_scale, slope_scale = activation64(activation, gate)
        close(read(inner)[:, 0], 2 * f, 32 * D.u * 2 * f_scale + 1e-37, 1.0, activation)
        blocks.gated_gemm_gradient(pre, None, D.tensor(np.ones((9, 1))), D.tensor(np.ones((1, 1))), pre, activation=activation)
        close(read(pre)[:, 0], 2 * slope, 32 * D.u * 2 * slope_scale + 1e-37, 1.0, activation)
        for rows in (9, 300):
            data = np.ones((rows, 40))
            data[3, 5] = np.nan
            inner = D.tensor(np.zeros((rows, 40)))
            blocks.gated_gemm(inner, None, D.tensor(data), D.tensor(np.ones((80, 40)) / 40), activation=activation)
            got = read(inner)
            assert np.all(np.isnan(got[3])) and np.all(np.isfinite(np.delete(got, 3, 0))), activation


def test_floats_beyond_the_pieces_range(stream):  # noqa: F811
    """Elements of 2^112 and more are multiplied as floats."""
    D = Owned("float")
    x = np.full((200, 64), 2.0 ** 115, np.float32)
    weights = np.full((300, 64), 2.0 ** -116, np.float32)
    inner, pre = D.tensor(np.zeros((200, 150))), D.tensor(np.zeros((200, 300)))
    blocks.gated_gemm(inner, pre, D.tensor(x), D.tensor(weights), activation="relu")
    assert np.all(read(pre) == 32.0) and np.all(read(inner) == 1024.0)
    D.free()


@pytest.mark.parametrize("datatype", ["float", "double"])
def test_recorded_into_a_graph(as_released, datatype):  # noqa: F811
    from test_gpu_graph_capture import hip_runtime
    rt = hip_runtime()
    stream = drv.HipDriver().default_device().create_stream()  # noqa: F811
    D = Owned(datatype)
    rng = np.random.default_rng(3)
    tokens, width, hidden = 48, 96, 80
    with ct.tensor_context(stream, datatype):
        block = blocks.GatedBlock(tokens, width, hidden, datatype=datatype)
        p = {k: {"buffer": D.tensor(rng.standard_normal(s) * 0.1), "gradient": D.tensor(np.zeros(s))}
             for k, s in (("first", (2 * hidden, width)), ("second", (width, hidden)), ("post-scale", (width,)), ("pre-scale", (width,)))}
        x, residual, output, normalized, dx, dr, dn = (D.tensor(np.zeros((tokens, width))) for _ in range(7))

        def once():
            block.forward(p, x, residual, output, normalized)
            block.backward(p, x, output, dx, dr, None, normalized)
            return None

        def results():
            return [read(t) for t in (output, dx, dr, p["first"]["gradient"], p["second"]["gradient"])]

        once()
        stream.sync()
        graph, executable = C.c_void_p(), C.c_void_p()
        assert rt.hipStreamBeginCapture(stream.handle, 1) == 0
        try:
            once()
        finally:
            ended = rt.hipStreamEndCapture(stream.handle, C.byref(graph))
        assert ended == 0 and graph.value
        assert rt.hipGraphInstantiate(C.byref(executable), graph, None, None, 0) == 0
        for _ in range(3):
            for t in (x, residual):
                ct.assign(t, D.tensor(rng.standard_normal((tokens, width))))
            once()
            eager = results()
            assert rt.hipGraphLaunch(executable, stream.handle) == 0
            assert all(np.array_equal(a, b) for a, b in zip(eager, results()))
        assert rt.hipGraphExecDestroy(executable) == 0 and rt.hipGraphDestroy(graph) == 0
    D.free()
    stream.release()


# ------------------------------------------------------------------------------------------------- the layers

def made(rng, shapes):
    return {k: rng.standard_normal(s) * scale + shift for k, (s, scale, shift) in shapes.items()}


def on_device(host, datatype):
    return {k: {"buffer": ct.to_tensor(v, datatype), "gradient": ct.new_tensor(list(v.shape), datatype=datatype)} for k, v in host.items()}


@pytest.mark.parametrize("activation", ["swish", "gelu", "tanh", "logistic"])
@pytest.mark.parametrize("experts", [None, 5])
def test_a_block_s_gradients_are_the_differences(stream, experts, activation):  # noqa: F811
    """In double: central differences of step 1e-5 along one direction through every parameter and input, bar 1e-6.  The choice of
    experts does not change over such a step for these inputs."""
    rng = np.random.default_rng(3)
    tokens, width, hidden = 13, 24, 40
    groups = () if experts is None else (experts,)
    shapes = {"first": ((*groups, 2 * hidden, width), width ** -0.5, 0.0), "second": ((*groups, width, hidden), hidden ** -0.5, 0.0),
              "post-scale": ((width,), 0.1, 1.0), "pre-scale": ((width,), 0.1, 1.0), "gate": ((1, width), 0.1, 0.5),
              "x": ((tokens, width), 1.0, 0.0), "residual": ((tokens, width), 1.0, 0.0)}
    if experts is not None:
        shapes["router"] = ((experts, width), 1.0, 0.0)
    host = made(rng, shapes)
    direction = {k: rng.standard_normal(v.shape) for k, v in host.items()}
    to_output, to_normalized = rng.standard_normal((tokens, width)), rng.standard_normal((tokens, width))
    with ct.tensor_context(stream, "double"):
        descriptor = blocks.norm_descriptor(residual_scale=0.8)
        block = (blocks.GatedBlock(tokens, width, hidden, descriptor, activation=activation) if experts is None else
                 blocks.ExpertBlock(tokens, width, hidden, experts, 2, descriptor, gated=activation))
        output, normalized = ct.new_tensor([tokens, width]), ct.new_tensor([tokens, width])
        values = lambda t: ct.to_double_array(t).reshape(t.shape())

        def value(step):
            p = on_device({k: v + step * direction[k] for k, v in host.items()}, "double")
            x, residual = p.pop("x"), p.pop("residual")
            block.forward(p, x["buffer"], residual["buffer"], output, normalized)
            return (values(output) * to_output).sum() + (values(normalized) * to_normalized).sum(), p, x, residual

        high, low = value(1e-5)[0], value(-1e-5)[0]
        _, p, x, residual = value(0.0)
        block.backward(p, x["buffer"], output, x["gradient"], residual["gradient"], ct.to_tensor(to_output), ct.to_tensor(to_normalized))
        p.update(x=x, residual=residual)
        along = sum((values(p[k]["gradient"]) * direction[k]).sum() for k in p)
        assert abs(along - (high - low) / 2e-5) <= 1e-6 * max(1.0, abs(along))
        for k in p:     # each parameter by itself
            assert np.linalg.norm(values(p[k]["gradient"])) > 0, k


@pytest.mark.parametrize("experts", [None, 4])
def test_training_steps_of_both_operators(as_released, experts):  # noqa: F811
    """Gated blocks whose matrices the orthogonalised step trains and whose vectors Adam does, after clipping: parameters without a
    gradient stay as they are, the others move by what the step allows."""
    stream = drv.HipDriver().default_device().create_stream()  # noqa: F811
    rng = np.random.default_rng(4)
    tokens, width, hidden = 96, 40, 56
    groups = () if experts is None else (experts,)
    shapes = {"first": ((*groups, 2 * hidden, width), width ** -0.5, 0.0), "second": ((*groups, width, hidden), hidden ** -0.5, 0.0),
              "post-scale": ((width,), 0.1, 1.0), "pre-scale": ((width,), 0.1, 1.0)}
    if experts is not None:
        shapes["router"] = ((experts, width), 1.0, 0.0)
    with ct.tensor_context(stream, "float"):
        p = on_device(made(rng, shapes), "float")
        block = (blocks.GatedBlock(tokens, width, hidden) if experts is None else blocks.ExpertBlock(tokens, width, hidden, experts, 2, gated="swish"))
        x, target = (ct.to_tensor(rng.standard_normal((tokens, width))) for _ in range(2))
        output, normalized, dx, dr, difference = (ct.new_tensor([tokens, width]) for _ in range(5))
        backend = optimize.Backend(stream, "float")
        matrices, vectors = optimize.create_optimizer(backend, optimize.muon(alpha=0.02)), optimize.create_optimizer(backend, optimize.adam())
        momentum = {k: {"momentum-vals": ct.new_tensor([v["buffer"].ecount()])} for k, v in p.items() if len(v["buffer"].shape()) > 1}
        memory = {"m": ct.new_tensor([2 * width]), "v": ct.new_tensor([2 * width])}
        norm = ct.new_tensor([2])
        p["pre-scale"]["gradient"] = None
        held = ct.to_double_array(p["pre-scale"]["buffer"])
        for _ in range(3):
            block.forward(p, x, x, output, normalized)
            ct.binary_op(difference, 1.0, normalized, 1.0, target, "-")
            block.backward(p, x, output, dx, dr, None, difference)
            optimize.clip_gradients(backend, [v["gradient"] for v in p.values() if v["gradient"] is not None], 1.0, norm)
            vectors, before = vectors.batch_update(), {k: ct.to_double_array(p[k]["buffer"]) for k in momentum}
            vectors.compute_parameters(memory, 1.0, 0, p["post-scale"]["gradient"], p["post-scale"]["buffer"])
            for k, state in momentum.items():
                matrices.compute_parameters(state, 1.0, 0, p[k]["gradient"], p[k]["buffer"])
                shape = p[k]["buffer"].shape()
                rate = 0.02 * max(1, shape[-2] / shape[-1]) ** 0.5
                moved = (ct.to_double_array(p[k]["buffer"]) - before[k]).reshape(-1, *shape[-2:])
                for m in moved:     # singular values of an orthogonalised matrix are below 1.3
                    assert 0 < np.linalg.norm(m, 2) <= 1.3 * rate, k
        assert np.array_equal(ct.to_double_array(p["pre-scale"]["buffer"]), held)
    stream.release()


def test_a_block_that_only_answers(stream):  # noqa: F811
    rng = np.random.default_rng(5)
    tokens, width, hidden = 3, 32, 48
    host = made(rng, {"first": ((2 * hidden, width), 0.2, 0.0), "second": ((width, hidden), 0.2, 0.0), "post-scale": ((width,), 0.1, 1.0)})
    with ct.tensor_context(stream, "float"):
        p = on_device(host, "float")
        x = ct.to_tensor(rng.standard_normal((tokens, width)))
        results = []
        for training in (True, False):
            block = blocks.GatedBlock(tokens, width, hidden, training=training)
            output, normalized = ct.new_tensor([tokens, width]), ct.new_tensor([tokens, width])
            block.forward(p, x, x, output, normalized)
            results.append((ct.to_double_array(output), ct.to_double_array(normalized)))
        assert all(np.array_equal(a, b) for a, b in zip(*results))
        with pytest.raises(ct.TensorError, match="not for training"):
            block.backward(p, x, output, x, x, None, x)
