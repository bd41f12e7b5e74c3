"""Matrices made orthogonal, and the optimizer step made of it, against their formulas in 64 bits (numpy).

Bars, fixed ahead.  With u = 2^-24 (float) or 2^-53 (double), a product of the library differs from the exact one by at most
(16 + 3 k / 16) u of the sum of its terms' magnitudes: an element is held to 2 u, what two pieces leave out of a product is 4 u, a result
is stored to 2 u, and a float sum rounds three times for 16 k (of which the signs differ: the root of their number is what is
seen, and the bars below take that).  The steps magnify such differences by what the matrix's singular values make of them, so the bar
of several steps is found in 64 bits: six times what the result moves by, in the root of the sum of squares, if after each product
normal noise of (8 + sqrt(k) / 2) u of the magnitudes is added.  One step's is found the same way and is also held to the proven bound.
"""
import ctypes as C
import threading

import numpy as np
import pytest

from cortex_amd import capi
from cortex_amd import driver as drv
from cortex_amd import optimize
from cortex_amd import tensor as ct
from test_gpu_blocks import NUMPY, UNIT, Owned, as_released, read, stream  # noqa: F401

pytestmark = pytest.mark.gpu

COEFFICIENTS = optimize.NEWTON_SCHULZ_COEFFICIENTS
MILD = (1.5, -0.5, 0.0)     # the step of third degree


def orthogonal64(g, steps=5, coefficients=COEFFICIENTS, epsilon=1e-7, noise=0.0, rng=None):
    g = np.asarray(g, np.float64)
    x = g / (np.sqrt((g * g).sum()) + epsilon)
    if x.shape[0] > x.shape[1]:
        x = x.T
    triples = coefficients if np.ndim(coefficients) == 2 else [coefficients] * steps

    def product(l, r):
        c = l @ r
        return c if not noise else c + noise * (8 + np.sqrt(l.shape[1]) / 2) * rng.standard_normal(c.shape) * (abs(l) @ abs(r))

    for a, b, c in triples:
        gram = product(x, x.T)
        x = product(a * np.eye(len(x)) + b * gram + c * product(gram, gram), x)
    return x.T if g.shape[0] > g.shape[1] else x


def bar_of(g, u, **kwargs):
    rng = np.random.default_rng(5)
    exact = orthogonal64(g, **kwargs)
    moved = max(np.linalg.norm(orthogonal64(g, noise=u, rng=rng, **kwargs) - exact) for _ in range(3))
    return exact, 6 * moved


def near(got, want, bar, what=""):
    assert np.all(np.isfinite(got)), what
    off = np.linalg.norm(np.asarray(got, np.float64) - want)
    assert off <= bar, f"{what}: {off:.3g} from {np.linalg.norm(want):.3g}, {off / bar:.3g} times the bar"


def gradient(rng, *shape):
    """A few directions and noise, as gradients are."""
    count, rows, columns = shape
    rank = max(1, min(rows, columns) // 8)
    return 1e-3 * (rng.standard_normal((count, rows, rank)) @ rng.standard_normal((count, rank, columns)) + 0.2 * rng.standard_normal(shape))


@pytest.fixture(params=["float", "double"])
def D(request, stream):  # noqa: F811
    owned = Owned(request.param)
    owned.u, owned.type = UNIT[request.param], NUMPY[request.param]
    owned.backend = optimize.Backend(stream, request.param)
    yield owned
    owned.free()


SHAPES = [(1, 1, 1), (1, 1, 7), (2, 7, 1), (1, 2, 2), (3, 5, 3), (1, 10, 128), (1, 32, 32), (2, 33, 31), (1, 64, 65), (4, 31, 97), (1, 100, 257),
          (1, 128, 784), (1, 257, 129), (2, 256, 256), (1, 300, 700), (1, 513, 130)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("steps", [1, 5])
def test_against_the_formula(D, shape, steps):
    rng = np.random.default_rng(hash(shape) % 1000)
    g = D.tensor(gradient(rng, *shape))
    out = D.tensor(np.full(shape, np.nan))
    workspace = optimize.orthogonalize_workspace(D.backend, g)
    optimize.orthogonalize(D.backend, out, g, steps=steps, workspace=workspace)
    values, got = read(g), read(out)
    for i in range(shape[0]):
        want, bar = bar_of(values[i], D.u, steps=steps)
        near(got[i], want, bar, f"matrix {i}")
        if steps == 1:
            m, n = sorted(shape[1:])
            c = lambda k: 16 + 3 * k / 16
            near(got[i], want, (9 * c(n) + 13 * c(m) + 7 * np.sqrt(m) + 32) * D.u, "the proven bound")
    workspace.release()


@pytest.mark.parametrize("shape", [(1, 900, 1100), (3, 640, 1280), (1, 2100, 520)], ids=str)
def test_larger(D, shape):
    rng = np.random.default_rng(3)
    g, out = D.tensor(gradient(rng, *shape)), D.tensor(np.zeros(shape))
    optimize.orthogonalize(D.backend, out, g, steps=3)
    values, got = read(g), read(out)
    for i in range(shape[0]):
        want, bar = bar_of(values[i], D.u, steps=3)
        near(got[i], want, bar)


def test_every_tile(stream, as_released):  # noqa: F811
    """Matrices that each side of tiles is taken for, many of one shape: each is its own."""
    D = Owned("float")
    backend = optimize.Backend(stream, "float")
    rng = np.random.default_rng(8)
    for shape in ((40, 70, 200), (24, 400, 300), (28, 760, 1000), (20, 1100, 1030)):
        one = gradient(rng, 1, *shape[1:])
        scales = 2.0 ** rng.integers(-3, 4, shape[0])      # a power of two in front changes no bit but for epsilon
        g, out = D.tensor(one * scales[:, None, None]), D.tensor(np.zeros(shape))
        optimize.orthogonalize(backend, out, g, steps=2, epsilon=0.0)
        got = read(out)
        want, bar = bar_of(read(g)[0], UNIT["float"], steps=2, epsilon=0.0)
        near(got[0], want, bar, shape)
        assert np.array_equal(got, np.broadcast_to(got[0], shape)), shape
        D.free()
        D.kept.clear()


@pytest.mark.parametrize("shape", [(14, 500, 600), (14, 600, 500), (3, 70, 3000), (2, 3000, 70), (1, 33, 1029), (2, 1029, 20), (1, 5, 65), (1, 130, 16), (1, 1, 5000)],
                         ids=str)
def test_every_kernel_of_doubles(stream, as_released, shape):  # noqa: F811
    """Tiles of 64 and of 32 for each product, and X X^T in parts of k; matrices that are powers of two apart have the same results."""
    D = Owned("double")
    rng = np.random.default_rng(31)
    one = gradient(rng, 1, *shape[1:])
    scales = 2.0 ** rng.integers(-3, 4, shape[0])
    g, out = D.tensor(one * scales[:, None, None]), D.tensor(np.full(shape, np.nan))
    optimize.orthogonalize(optimize.Backend(stream, "double"), out, g, steps=3, epsilon=0.0)
    got = read(out)
    want, bar = bar_of(one[0], UNIT["double"], steps=3, epsilon=0.0)
    near(got[0], want, bar)
    assert np.array_equal(got, np.broadcast_to(got[0], shape))
    D.free()


@pytest.mark.parametrize("rows,columns", [(37, 65), (65, 37), (1, 9), (9, 1)])
def test_rows_apart_and_what_the_result_is_added_to(D, rows, columns):
    rng = np.random.default_rng(1)
    g = D.block(gradient(rng, 1, rows, columns)[0], 3)
    before = rng.standard_normal((rows, columns)).astype(D.type)
    out = D.block(before, 5)
    optimize.orthogonalize(D.backend, out, g, alpha=-0.5, beta=0.25)
    want, bar = bar_of(read(g), D.u)
    near(read(out), 0.25 * before - 0.5 * want, 0.5 * bar + 4 * D.u * np.linalg.norm(before))


def test_in_place_and_in_turns(D):
    shape = (5, 33, 70)
    rng = np.random.default_rng(2)
    data = gradient(rng, *shape)
    g, out = D.tensor(data), D.tensor(np.zeros(shape))
    whole = optimize.orthogonalize_workspace(D.backend, g)
    optimize.orthogonalize(D.backend, out, g, workspace=whole)
    one = D.backend.stream.orthogonalize_workspace(1, *shape[1:], D.backend.datatype)
    # two at a time, the last by itself, into the input; what lies behind what the call was given stays as it is
    optimize.orthogonalize(D.backend, g, g, workspace=whole.sub_buffer(0, 2 * one + 100))
    assert np.array_equal(read(out), read(g))
    whole.release()


def test_values_at_the_ends_of_the_range(D):
    rng = np.random.default_rng(4)
    data = np.asarray(gradient(rng, 1, 48, 40)[0], D.type)
    u = D.u
    for scale in (2.0 ** -100, 2.0 ** 100) if D.type == np.float32 else (2.0 ** -400, 2.0 ** 400):
        g, out = D.tensor(data * D.type(scale)), D.tensor(np.zeros((48, 40)))
        optimize.orthogonalize(D.backend, out, g, epsilon=0.0)
        want, bar = bar_of(read(g) * (1 / scale), u, epsilon=0.0)
        near(read(out), want, bar, scale)
    # one singular value; rows of zeros; all zeros
    g = D.tensor(np.outer(rng.standard_normal(20), rng.standard_normal(33)))
    out = D.tensor(np.zeros((20, 33)))
    optimize.orthogonalize(D.backend, out, g)
    want, bar = bar_of(read(g), u)
    near(read(out), want, bar)
    data = np.asarray(gradient(rng, 1, 20, 33)[0])
    data[3:9] = 0
    g = D.tensor(data)
    optimize.orthogonalize(D.backend, out, g)
    want, bar = bar_of(read(g), u)
    near(read(out), want, bar)
    assert np.all(read(out)[3:9] == 0)
    optimize.orthogonalize(D.backend, out, D.tensor(np.zeros((20, 33))))
    assert np.all(read(out) == 0)


def test_what_is_not_finite_stays_in_its_matrix(D):
    rng = np.random.default_rng(6)
    data = gradient(rng, 3, 40, 70)
    clean, bad = D.tensor(data), data.copy()
    bad[1, 3, 5] = np.nan
    for value in (np.nan, np.inf, -np.inf):
        bad[1, 3, 5] = value
        g, out, want = D.tensor(bad), D.tensor(np.zeros((3, 40, 70))), D.tensor(np.zeros((3, 40, 70)))
        optimize.orthogonalize(D.backend, out, g)
        optimize.orthogonalize(D.backend, want, clean)
        got, want = read(out), read(want)
        assert np.all(np.isnan(got[1])), value
        assert np.array_equal(got[[0, 2]], want[[0, 2]]), value


@pytest.mark.parametrize("coefficients", [MILD, (2.0, -1.5, 0.5), (0.0, 0.0, 0.0), (-1.0, 0.0, 0.0), (40.0, 0.0, 0.0), (1e-3, 0.0, 0.0),
                                          [(4.0, -6.0, 2.5), (3.0, -3.5, 1.25), (1.5, -0.5, 0.0)]], ids=str)
def test_coefficients(D, coefficients):
    rng = np.random.default_rng(9)
    steps = 3
    g, out = D.tensor(gradient(rng, 2, 60, 44)), D.tensor(np.zeros((2, 60, 44)))
    optimize.orthogonalize(D.backend, out, g, steps=steps, coefficients=coefficients)
    for i in range(2):
        want, bar = bar_of(read(g)[i], D.u, steps=steps, coefficients=coefficients)
        near(read(out)[i], want, bar + 16 * D.u * np.linalg.norm(want))


@pytest.mark.parametrize("shape", [(1, 3, 2000), (2, 2000, 3), (2, 16, 129), (3, 17, 1000), (1, 1000, 17), (2, 48, 300), (1, 300, 48), (2, 49, 70), (1, 64, 5001),
                                   (2, 5001, 64), (5, 64, 64)], ids=str)
def test_few_rows(D, shape):
    """Added to what is there, rows apart."""
    rng = np.random.default_rng(20)
    count, rows, columns = shape
    whole, target = rng.standard_normal((count, rows, columns + 5)), rng.standard_normal((count, rows, columns + 3))
    whole[:, :, :columns] = gradient(rng, *shape)
    g, out = D.tensor(whole), D.tensor(target)
    before, values = read(out), read(g)
    need = D.backend.stream.orthogonalize_workspace(count, rows, columns, D.backend.datatype)
    workspace = D.backend.stream.get_device().allocate_device_buffer(need, "byte")
    D.backend.stream.orthogonalize(optimize._buffer(out), columns + 3, rows * (columns + 3), 0.5, optimize._buffer(g), columns + 5, rows * (columns + 5), 0.25,
                                   count, rows, columns, optimize._steps_of(COEFFICIENTS, 5), 1e-7, workspace)
    got = read(out)
    workspace.release()
    assert np.array_equal(got[:, :, columns:], before[:, :, columns:])
    for i in range(count):
        want, bar = bar_of(values[i, :, :columns], D.u)
        want = 0.5 * want + 0.25 * before[i, :, :columns]
        near(got[i, :, :columns], want, 0.5 * bar + 4 * D.u * np.linalg.norm(abs(want) + abs(before[i, :, :columns])))


@pytest.mark.parametrize("steps", [5, 6, 7, 12, 25, 64])
@pytest.mark.parametrize("shape", [(20, 90), (90, 64), (100, 200)], ids=str)
def test_many_steps_of_a_singular_matrix(D, shape, steps):
    """Singular values of 0, which rounding makes others of: all stay below what the steps allow, 1.2024, and a little for rounding."""
    rng = np.random.default_rng(21)
    values = gradient(rng, 1, *shape)[0]
    values[: shape[0] // 2] = values[shape[0] // 2: 2 * (shape[0] // 2)]
    g, out = D.tensor(values), D.tensor(np.zeros(shape))
    optimize.orthogonalize(D.backend, out, g, steps=steps)
    got = read(out).astype(np.float64)
    assert np.all(np.isfinite(got)) and np.linalg.svd(got, compute_uv=False).max() < 1.21


def test_singular_values_end_near_one(D):
    rng = np.random.default_rng(10)
    g, out = D.tensor(rng.standard_normal((96, 200))), D.tensor(np.zeros((96, 200)))
    optimize.orthogonalize(D.backend, out, g, steps=12, coefficients=MILD)
    values = np.linalg.svd(read(out).astype(np.float64), compute_uv=False)
    assert np.all(abs(values - 1) < 0.3)
    optimize.orthogonalize(D.backend, out, g)
    values = np.linalg.svd(read(out).astype(np.float64), compute_uv=False)
    assert np.all((values > 0.6) & (values < 1.3))


def step64(g, p, v, o, alpha):
    g, p, v = (np.asarray(x, np.float64) for x in (g, p, v))
    v = o["momentum"] * v + alpha * g
    return v, alpha * g + o["momentum"] * v if o["nesterov"] else v


@pytest.mark.parametrize("shape", [(10, 128), (128, 784), (33, 20), (3, 40, 70), (2, 70, 40), (1, 1)], ids=str)
@pytest.mark.parametrize("nesterov,decay", [(True, 0.0), (False, 0.1)])
def test_step(D, shape, nesterov, decay):
    rng = np.random.default_rng(11)
    count, rows, columns = shape if len(shape) == 3 else (1, *shape)
    o = optimize.muon(alpha=0.05, nesterov=nesterov, **{"weight-decay": decay})
    optimizer = optimize.create_optimizer(D.backend, o)
    data = [np.asarray(x.reshape(shape), D.type) for x in (64 * gradient(rng, count, rows, columns), rng.standard_normal((count, rows, columns)))]
    g, p = map(D.tensor, data)
    n, offset = int(np.prod(shape)), 5
    state = {"momentum-vals": D.tensor(np.zeros(n + 2 * offset))}
    for step in range(2):
        before, v_before = read(p), read(state["momentum-vals"])
        optimizer.batch_update().compute_parameters(state, 1 / 64, offset, g, p)
        v, u = step64(data[0], before, v_before[offset:offset + n].reshape(shape), o, 1 / 64)
        whole = read(state["momentum-vals"])
        got = whole[offset:offset + n].reshape(shape)
        assert np.all(whole[:offset] == 0) and np.all(whole[offset + n:] == 0)
        assert np.all(abs(got - v) <= 4 * D.u * (abs(v) + abs(data[0]) / 64)), "momentum"
        rate = 0.05 * np.sqrt(max(1, rows / columns))
        for i in range(count):
            at = (lambda x: x.reshape(count, rows, columns)[i])
            want, bar = bar_of(at(u), D.u)
            near(at(read(p)), at(before) * (1 - 0.05 * decay) - rate * want, rate * bar + 4 * D.u * np.linalg.norm(at(before)), f"step {step}")


def test_nothing_to_do(D):
    for shape in ((0, 5), (5, 0), (0, 3, 4)):
        t = D.tensor(np.zeros(shape))
        optimize.orthogonalize(D.backend, t, t)
    out = D.tensor(np.ones((3, 0, 4)))
    optimize.create_optimizer(D.backend, optimize.muon()).compute_parameters({"momentum-vals": D.tensor(np.zeros(1))}, 1.0, 0, out, out)


def test_two_streams_and_threads(as_released):  # noqa: F811
    """Two threads, a stream and a workspace each."""
    device = drv.HipDriver().default_device()
    rng = np.random.default_rng(12)
    inputs = [gradient(rng, 1, 200, 300)[0].astype(np.float32) for _ in range(2)]
    results = [[], []]

    def work(i):
        s = device.create_stream()
        capi.call("ct_set_device", 0)
        with ct.tensor_context(s, "float"):
            backend = optimize.Backend(s, "float")
            g, out = ct.to_tensor(inputs[i]), ct.new_tensor([200, 300])
            workspace = optimize.orthogonalize_workspace(backend, g)
            for _ in range(20):
                optimize.orthogonalize(backend, out, g, workspace=workspace)
                results[i].append(ct.to_array_of_type(out, "float").reshape(200, 300).copy())
            workspace.release()
        s.release()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        want, bar = bar_of(inputs[i], UNIT["float"])
        near(results[i][0], want, bar)
        assert len(results[i]) == 20 and all(np.array_equal(r, results[i][0]) for r in results[i])


@pytest.mark.parametrize("datatype", ["float", "double"])
def test_recorded_into_a_graph(as_released, datatype):  # noqa: F811
    from test_gpu_graph_capture import hip_runtime
    rt = hip_runtime()
    stream = drv.HipDriver().default_device().create_stream()  # noqa: F811
    D = Owned(datatype)
    with ct.tensor_context(stream, datatype):
        backend = optimize.Backend(stream, datatype)
        rng = np.random.default_rng(13)
        g, p, v = (D.tensor(gradient(rng, 2, 70, 40)) for _ in range(3))
        state = {"momentum-vals": v}
        optimizer = optimize.create_optimizer(backend, optimize.muon())
        start = [read(t) for t in (g, p, v)]
        eager = []
        for _ in range(4):
            optimizer.compute_parameters(state, 1.0, 0, g, p)
            eager.append((read(p), read(v)))
        for t, x in zip((g, p, v), start):
            ct.assign(t, D.tensor(x))
        stream.sync()
        graph, executable = C.c_void_p(), C.c_void_p()
        assert rt.hipStreamBeginCapture(stream.handle, 1) == 0
        try:
            optimizer.compute_parameters(state, 1.0, 0, g, p)
        finally:
            ended = rt.hipStreamEndCapture(stream.handle, C.byref(graph))
        assert ended == 0 and graph.value
        assert rt.hipGraphInstantiate(C.byref(executable), graph, None, None, 0) == 0
        other = D.tensor(np.ones((300, 300)))
        for i in range(4):
            assert rt.hipGraphLaunch(executable, stream.handle) == 0
            got = read(p), read(v)
            assert np.array_equal(got[0], eager[i][0]) and np.array_equal(got[1], eager[i][1]), i
            optimize.orthogonalize(backend, other, other)      # between the replays, with a workspace of its own
        assert rt.hipGraphExecDestroy(executable) == 0 and rt.hipGraphDestroy(graph) == 0
    D.free()
    stream.release()
