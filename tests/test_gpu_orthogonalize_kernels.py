"""Matrices made orthogonal by each of the kernels that float ones with both sides above 64 take: named by the call, at sizes that the
choice among them takes them for; and there what test_gpu_orthogonalize checks of smaller matrices.  Bars as there.
"""
import ctypes as C

import numpy as np
import pytest

from cortex_amd import capi
from cortex_amd import driver as drv
from cortex_amd import optimize
from cortex_amd import tensor as ct
from test_gpu_blocks import UNIT, Owned, as_released, read, stream  # noqa: F401
from test_gpu_orthogonalize import COEFFICIENTS, MILD, bar_of, gradient, near, orthogonal64, step64

pytestmark = pytest.mark.gpu

U = UNIT["float"]


@pytest.fixture
def D(stream):  # noqa: F811
    owned = Owned("float")
    owned.backend = optimize.Backend(stream, "float")
    yield owned
    owned.free()


def taken():
    """The tiles of each product that the last call took."""
    words = capi.last_kernel().split()
    assert words[0] == "orthogonalize_pair", words
    return dict(zip(words[1::2], words[2::2]))


KERNELS = [
    ((3, 70, 3000), dict(gram="parts", square="32", update="64", result="64")),
    ((2, 3001, 70), dict(gram="parts")),
    ((1, 200, 8001), dict(gram="parts", square="32")),
    ((1, 1402, 71), dict(gram="parts")),
    ((5, 80, 110), dict(gram="32", square="32", update="32", result="32")),
    ((1, 513, 130), dict(gram="32", square="32", update="32", result="32")),
    ((27, 261, 186), dict(gram="64", square="64")),
    ((3, 640, 1281), dict(gram="64", square="64", update="64", result="64")),
    ((26, 93, 2362), dict(update="128", result="128")),
    ((12, 1245, 715), dict(gram="128", square="128")),
    ((12, 642, 1213), dict(gram="128", update="256", result="256")),
    ((10, 1654, 1201), dict(gram="256x192", square="256x192", update="128", result="128")),
    ((15, 957, 2155), dict(gram="256x192", square="64", update="128")),
    ((30, 752, 1249), dict(gram="256")),
    ((15, 1233, 1418), dict(gram="256", square="256", update="256", result="256")),
]


@pytest.mark.parametrize("shape,expected", KERNELS, ids=str)
def test_each_kernel_by_name(D, shape, expected):
    """Many matrices of one shape are powers of two apart, which changes no bit but for epsilon: one is compared with the formula, the
    others with it."""
    rng = np.random.default_rng(8)
    one = gradient(rng, 1, *shape[1:])
    scales = 2.0 ** rng.integers(-3, 4, shape[0])
    g, out = D.tensor(one * scales[:, None, None]), D.tensor(np.full(shape, np.nan))
    optimize.orthogonalize(D.backend, out, g, steps=3, epsilon=0.0)
    met = taken()
    assert all(met[k] == v for k, v in expected.items()), met
    got = read(out)
    want, bar = bar_of(read(g)[0], U, steps=3, epsilon=0.0)
    near(got[0], want, bar, shape)
    assert np.array_equal(got, np.broadcast_to(got[0], shape))


APART = [((2, 90, 130), "32"), ((2, 130, 90), "32"), ((3, 70, 1380), "64"), ((2, 1380, 71), "64"), ((26, 93, 2362), "128"), ((25, 2469, 113), "128"),
         ((33, 196, 1686), "256"), ((14, 1756, 470), "256")]


@pytest.mark.parametrize("shape,side", APART, ids=str)
def test_rows_apart_and_added_to_what_is_there(D, shape, side):
    rng = np.random.default_rng(20)
    count, rows, columns = shape
    whole, target = rng.standard_normal((count, rows, columns + 5)), rng.standard_normal((count, rows, columns + 3))
    whole[:, :, :columns] = gradient(rng, *shape)
    g, out = D.tensor(whole), D.tensor(target)
    before, values = read(out), read(g)
    workspace = D.backend.stream.get_device().allocate_device_buffer(D.backend.stream.orthogonalize_workspace(count, rows, columns, "float"), "byte")
    D.backend.stream.orthogonalize(optimize._buffer(out), columns + 3, rows * (columns + 3), 0.5, optimize._buffer(g), columns + 5, rows * (columns + 5), 0.25,
                                   count, rows, columns, optimize._steps_of(COEFFICIENTS, 3), 1e-7, workspace)
    assert taken()["result"] == side, taken()
    got = read(out)
    workspace.release()
    assert np.array_equal(got[:, :, columns:], before[:, :, columns:]) and np.array_equal(read(g), values)
    for i in sorted({0, count // 2, count - 1}):
        want, bar = bar_of(values[i, :, :columns], U, steps=3)
        want = 0.5 * want + 0.25 * before[i, :, :columns]
        near(got[i, :, :columns], want, 0.5 * bar + 4 * U * np.linalg.norm(abs(want) + abs(before[i, :, :columns])), i)


@pytest.mark.parametrize("shape", [(5, 80, 110), (5, 110, 80), (3, 70, 3000), (4, 300, 700)], ids=str)
def test_in_place_and_in_turns(D, shape):
    rng = np.random.default_rng(2)
    g, out = D.tensor(gradient(rng, *shape)), D.tensor(np.zeros(shape))
    one = D.backend.stream.orthogonalize_workspace(1, *shape[1:], "float")
    room = D.backend.stream.get_device().allocate_device_buffer(one * (shape[0] + 1), "byte")
    # two at a time, the last by itself, and one at a time: of fewer matrices at once other kernels may be taken, so each against the formula
    values = read(g)
    for at_once in (2, 1):
        optimize.orthogonalize(D.backend, out, g, workspace=room.sub_buffer(0, at_once * one + 100))
        got = read(out)
        for i in range(shape[0]):
            want, bar = bar_of(values[i], U)
            near(got[i], want, bar, (at_once, i))
    optimize.orthogonalize(D.backend, g, g, workspace=room.sub_buffer(0, one))
    assert taken()["result"] != ""
    assert np.array_equal(read(g), got)
    room.release()


@pytest.mark.parametrize("shape", [(70, 130), (130, 70), (300, 400), (70, 2500)], ids=str)
def test_values_at_the_ends_of_the_range(D, shape):
    rng = np.random.default_rng(4)
    data = np.asarray(gradient(rng, 1, *shape)[0], np.float32)
    want, bar = bar_of(data, U, epsilon=0.0)
    out = D.tensor(np.zeros(shape))
    for scale in (2.0 ** -100, 2.0 ** 100):
        optimize.orthogonalize(D.backend, out, D.tensor(data * np.float32(scale)), epsilon=0.0)
        taken()
        near(read(out), want, bar, scale)
    # one singular value; rows and columns of zeros; all zeros
    g = D.tensor(np.outer(rng.standard_normal(shape[0]), rng.standard_normal(shape[1])))
    optimize.orthogonalize(D.backend, out, g)
    want, bar = bar_of(read(g), U)
    near(read(out), want, bar)
    data = np.asarray(gradient(rng, 1, *shape)[0])
    data[3:9], data[:, 20:33] = 0, 0
    g = D.tensor(data)
    optimize.orthogonalize(D.backend, out, g)
    want, bar = bar_of(read(g), U)
    near(read(out), want, bar)
    assert np.all(read(out)[3:9] == 0) and np.all(read(out)[:, 20:33] == 0)
    optimize.orthogonalize(D.backend, out, D.tensor(np.zeros(shape)))
    assert np.all(read(out) == 0)


@pytest.mark.parametrize("shape", [(3, 70, 130), (3, 130, 70), (3, 300, 400), (3, 70, 2500), (26, 93, 2362)], ids=str)
def test_what_is_not_finite_stays_in_its_matrix(D, shape):
    rng = np.random.default_rng(6)
    data = gradient(rng, *shape)
    clean, bad = D.tensor(data), data.copy()
    want, out = D.tensor(np.zeros(shape)), D.tensor(np.zeros(shape))
    optimize.orthogonalize(D.backend, want, clean)
    want = read(want)
    others = [i for i in range(shape[0]) if i != 1]
    for value in (np.nan, np.inf, -np.inf):
        bad[1, 3, 5] = value
        optimize.orthogonalize(D.backend, out, D.tensor(bad))
        taken()
        got = read(out)
        assert np.all(np.isnan(got[1])), value
        assert np.array_equal(got[others], want[others]), value


@pytest.mark.parametrize("coefficients", [MILD, (2.0, -1.5, 0.5), (0.0, 0.0, 0.0), (-1.0, 0.0, 0.0), (40.0, 0.0, 0.0), (1e-3, 0.0, 0.0),
                                          [(4.0, -6.0, 2.5), (3.0, -3.5, 1.25), (1.5, -0.5, 0.0)]], ids=str)
@pytest.mark.parametrize("shape", [(2, 90, 70), (1, 260, 300)], ids=str)
def test_coefficients(D, shape, coefficients):
    rng = np.random.default_rng(9)
    g, out = D.tensor(gradient(rng, *shape)), D.tensor(np.zeros(shape))
    optimize.orthogonalize(D.backend, out, g, steps=3, coefficients=coefficients)
    taken()
    for i in range(shape[0]):
        want, bar = bar_of(read(g)[i], U, steps=3, coefficients=coefficients)
        near(read(out)[i], want, bar + 16 * U * np.linalg.norm(want))


@pytest.mark.parametrize("shape", [(300, 500), (500, 300), (2, 400, 110), (26, 93, 2362)], ids=str)
@pytest.mark.parametrize("nesterov,decay", [(True, 0.0), (False, 0.1)])
def test_step(D, shape, nesterov, decay):
    rng = np.random.default_rng(11)
    count, rows, columns = shape if len(shape) == 3 else (1, *shape)
    o = optimize.muon(alpha=0.05, nesterov=nesterov, **{"weight-decay": decay})
    optimizer = optimize.create_optimizer(D.backend, o)
    data = [np.asarray(x.reshape(shape), np.float32) for x in (64 * gradient(rng, count, rows, columns), rng.standard_normal((count, rows, columns)))]
    g, p = map(D.tensor, data)
    n, offset = int(np.prod(shape)), 5
    state = {"momentum-vals": D.tensor(np.zeros(n + 2 * offset))}
    for step in range(2):
        before, v_before = read(p), read(state["momentum-vals"])
        optimizer.batch_update().compute_parameters(state, 1 / 64, offset, g, p)
        taken()
        v, u = step64(data[0], before, v_before[offset:offset + n].reshape(shape), o, 1 / 64)
        whole = read(state["momentum-vals"])
        assert np.all(whole[:offset] == 0) and np.all(whole[offset + n:] == 0)
        assert np.all(abs(whole[offset:offset + n].reshape(shape) - v) <= 4 * U * (abs(v) + abs(data[0]) / 64)), "momentum"
        rate = 0.05 * np.sqrt(max(1, rows / columns))
        for i in sorted({0, count // 2, count - 1}):
            at = (lambda x: x.reshape(count, rows, columns)[i])
            want, bar = bar_of(at(u), U)
            near(at(read(p)), at(before) * (1 - 0.05 * decay) - rate * want, rate * bar + 4 * U * np.linalg.norm(at(before)), f"step {step}")


@pytest.mark.parametrize("shape", [(2, 90, 70), (1, 70, 2500), (1, 300, 500)], ids=str)
def test_recorded_into_a_graph(as_released, shape):  # noqa: F811
    from test_gpu_graph_capture import hip_runtime
    rt = hip_runtime()
    stream = drv.HipDriver().default_device().create_stream()  # noqa: F811
    D = Owned("float")
    with ct.tensor_context(stream, "float"):
        backend = optimize.Backend(stream, "float")
        rng = np.random.default_rng(13)
        g, p, v = (D.tensor(gradient(rng, *shape)) for _ in range(3))
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


def bars_of(g, u, **kwargs):
    """As bar_of, of each row and of each column by itself."""
    rng = np.random.default_rng(5)
    exact = orthogonal64(g, **kwargs)
    moved = [orthogonal64(g, noise=u, rng=rng, **kwargs) - exact for _ in range(3)]
    return exact, [6 * np.max([np.linalg.norm(x, axis=axis) for x in moved], axis=0) for axis in (1, 0)]


MAGNITUDES = [(1, 200, 400), (1, 400, 200), (3, 640, 700), (1, 70, 3000), (2, 3001, 70), (26, 93, 2362), (12, 1245, 715), (30, 752, 1249), (15, 957, 2155)]


@pytest.mark.parametrize("steps", [1, 5])
@pytest.mark.parametrize("of", ["rows", "columns", "both"])
@pytest.mark.parametrize("shape", MAGNITUDES, ids=str)
def test_rows_and_columns_of_unlike_magnitudes(D, shape, of, steps):
    """Rows of outputs, or columns of features, that are seldom used: each is held to a float's bits of itself, as products of floats hold it.  With
    the bars of the other tests, row by row and column by column; noise of the terms' magnitudes is as small as the row."""
    rng = np.random.default_rng(41)
    count, rows, columns = shape
    one = rng.standard_normal((rows, columns))
    if of != "columns":
        one *= 2.0 ** -rng.integers(0, 40, (rows, 1))
    if of != "rows":
        one *= 2.0 ** -rng.integers(0, 40, (1, columns))
    g, out = D.tensor(np.broadcast_to(one, shape)), D.tensor(np.zeros(shape))
    optimize.orthogonalize(D.backend, out, g, steps=steps)
    taken()
    got = read(out)
    want, bars = bars_of(read(g)[0], U, steps=steps)
    assert np.all(np.isfinite(got))
    for bar, axis in zip(bars, (1, 0)):
        off = np.linalg.norm(got[0] - want, axis=axis) / bar
        assert np.all(off <= 1), (("row", "column")[axis == 0], int(off.argmax()), float(off.max()))
    assert np.array_equal(got, np.broadcast_to(got[0], shape))


def test_magnitudes_over_the_whole_range(D):
    """Rows from 2^100 down to the least numbers: what the largest ones leave of the others is a float, or 0."""
    rng = np.random.default_rng(42)
    for shape in ((130, 300), (300, 130)):
        data = rng.standard_normal(shape)
        short = 0 if shape[0] < shape[1] else 1
        data *= np.expand_dims(2.0 ** np.linspace(100, -145, shape[short]), 1 - short)
        g, out = D.tensor(data), D.tensor(np.zeros(shape))
        optimize.orthogonalize(D.backend, out, g, epsilon=0.0)
        taken()
        want, bars = bars_of(read(g), U, epsilon=0.0)
        got = read(out)
        assert np.all(np.isfinite(got))
        off = np.linalg.norm(got - want, axis=1 - short)
        assert np.all(off <= bars[short] + 2.0 ** -149 * np.sqrt(max(shape)))


def test_memory_that_is_refused(D):
    """A step whose workspace there is no memory for takes a smaller one, and neither it nor what follows reports the refusal."""
    device, shape = D.backend.stream.get_device(), (6, 90, 70)
    one = D.backend.stream.orthogonalize_workspace(1, *shape[1:], "float")

    class Little:
        def allocate_device_buffer(self, n, datatype):
            return device.allocate_device_buffer(n if n <= one else 1 << 50, datatype)

    class Stream:
        def __getattr__(self, name):
            return getattr(D.backend.stream, name)

        def get_device(self):
            return Little()

    results = []
    for stream in (D.backend.stream, Stream()):
        data = [np.asarray(gradient(np.random.default_rng(i), *shape), np.float32) for i in range(3)]
        g, p, v = map(D.tensor, data)
        optimizer = optimize.create_optimizer(optimize.Backend(stream, "float"), optimize.muon())
        for _ in range(2):
            optimizer.compute_parameters({"momentum-vals": v}, 1.0, 0, g, p)
        results.append((read(p), read(v)))
        assert [w.ecount() for w in optimizer._workspaces] == [one if stream is not D.backend.stream else 6 * one]
    assert np.array_equal(results[0][1], results[1][1])
    for i in range(shape[0]):     # other tiles: sums in another order, 150 half steps of a float cover twice the bar of either
        assert np.linalg.norm(results[0][0][i] - results[1][0][i]) <= 150 * U * np.linalg.norm(results[0][0][i])


@pytest.mark.parametrize("shape", [(48, 40), (130, 300), (3, 3000)], ids=str)
def test_doubles_whose_squares_are_none(stream, shape):  # noqa: F811
    """The norm of matrices of which squares overflow, or vanish: powers of two apart they have the same results."""
    D = Owned("double")
    backend = optimize.Backend(stream, "double")
    rng = np.random.default_rng(52)
    data = gradient(rng, 1, *shape)[0]
    want, bar = bar_of(data, UNIT["double"], epsilon=0.0)
    out = D.tensor(np.zeros(shape))
    for exponent in (-980, -600, -490, 490, 600, 1015):
        optimize.orthogonalize(backend, out, D.tensor(np.ldexp(data, exponent)), epsilon=0.0)
        near(read(out), want, bar, exponent)
    # some of each kind: the large ones' norm, to which the others still belong
    for exponent in (-480, 475, 480, 485):
        mixed = data * 2.0 ** rng.integers(-12, 13, shape[0])[:, None]
        want, bar = bar_of(mixed, UNIT["double"], epsilon=0.0)
        optimize.orthogonalize(backend, out, D.tensor(np.ldexp(mixed, exponent)), epsilon=0.0)
        near(read(out), want, bar, exponent)
    # epsilon is added to the norm as it is
    for exponent in (-500, 500):
        optimize.orthogonalize(backend, out, D.tensor(np.ldexp(data, exponent)), epsilon=float(np.ldexp(np.linalg.norm(data), exponent)))
        want, bar = bar_of(data, UNIT["double"], epsilon=np.linalg.norm(data))
        near(read(out), want, bar, ("epsilon", exponent))
    optimize.orthogonalize(backend, out, D.tensor(np.ldexp(data, -1000)))     # 1e-7 beside which the norm is nothing
    assert np.all(abs(read(out)) <= 1e-290)
    D.free()
