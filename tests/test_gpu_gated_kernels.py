"""The gated products' kernels, each at a size that the choice among them takes it for: named by the call, and against the formulas in
64 bits with the bars of test_gpu_gated.
"""
import numpy as np
import pytest

from cortex_amd import blocks
from cortex_amd import capi
from test_gpu_blocks import NUMPY, UNIT, Owned, close, read, stream  # noqa: F401
from test_gpu_gated import check

pytestmark = pytest.mark.gpu


def owned(datatype):
    D = Owned(datatype)
    D.u, D.type = UNIT[datatype], NUMPY[datatype]
    return D


DOUBLE_TILES = [
    # (rows, width, hidden, groups), what forward and gradient take
    ((2177, 17, 183), {}, "gated_double_tiles", None),
    ((1001, 701, 901), {"activation": "gelu"}, "gated_double_tiles", None),
    ((1001, 701, 901), {"pad": 3, "keep": False}, "gated_double_tiles", None),
    ((1290, 1967, 1468), {}, "gated_double_tiles", "gated_gradient_double_tiles"),
    ((942, 19, 455, 3), {"indexed": True, "kind": "gaps"}, "gated_double_tiles", None),
    ((1102, 593, 3403, 3), {"indexed": True, "kind": "gaps", "activation": "tanh"}, "gated_double_tiles", "gated_gradient_double_tiles"),
    ((961, 955, 2907, 8), {"indexed": True}, "gated_double_tiles", "gated_gradient_double_tiles"),
    ((231, 7417, 731), {}, "gated_double_tiles+gated_sum", None),
    ((285, 6753, 367, 8), {"indexed": True, "kind": "gaps"}, "gated_double_tiles+gated_sum", None),
    ((2159, 4479, 671), {"activation": "logistic"}, None, "gated_gradient_double_tiles+gated_sum"),
]


@pytest.mark.parametrize("size,kwargs,forward,gradient", DOUBLE_TILES, ids=lambda x: str(x))
def test_tiles_of_64_doubles(stream, size, kwargs, forward, gradient):  # noqa: F811
    """Gates and ups that meet in LDS, rows by index with absent ones, parts of k, and the gradient in place (each call of `check`)."""
    D = owned("double")
    met = check(D, *size, seed=1, **kwargs)
    assert forward is None or met[0] == forward, met
    assert gradient is None or met[1] == gradient, met
    D.free()


FLOATS = [
    ((1, 33, 9), {}, "gated_thin", "gated_gradient_thin"),
    ((3, 1071, 25), {}, "gated_thin_long", "gated_gradient_thin_long"),
    ((2, 1153, 30, 8), {"indexed": True, "kind": "gaps"}, "gated_thin_long", "gated_gradient_thin_long"),
    ((7, 27, 1379, 8), {}, "gated_thin_wide", None),
    ((9, 37, 3306, 8), {"indexed": True, "kind": "gaps"}, "gated_thin_wide", "gated_gradient_thin_wide"),
    ((14, 70, 3210, 8), {"pad": 1}, "gated_thin_wide", "gated_gradient_thin_wide"),
    ((6, 3167, 1058, 8), {}, "gated_thin_wide_long", None),
    ((5, 3718, 2387, 8), {"indexed": True}, "gated_thin_wide_long", "gated_gradient_thin_wide_long"),
    ((7, 2483, 1722, 8), {"kind": "gaps", "activation": "gelu"}, None, "gated_gradient_thin_wide_long"),
    ((407, 49, 1081), {}, "gated_medium", None),
    ((1016, 63, 680), {}, None, "gated_gradient_medium"),
    ((844, 57, 927, 8), {"indexed": True, "kind": "gaps"}, None, "gated_gradient_medium"),
    ((81, 6822, 249), {}, "gated_medium+gated_sum", None),
    ((23, 3363, 3728), {}, None, "gated_gradient_medium+gated_sum"),
    ((342, 54, 3319, 3), {"indexed": True}, "gated_large", None),
    ((616, 36, 3535, 8), {"kind": "gaps"}, None, "gated_gradient_large"),
    ((89, 4870, 972), {}, "gated_large+gated_sum", None),
    ((196, 1542, 1330, 3), {"indexed": True, "kind": "gaps"}, "gated_large+gated_sum", None),
    ((795, 2326, 493), {}, None, "gated_gradient_large+gated_sum"),
    ((565, 1760, 883, 8), {"kind": "gaps"}, None, "gated_gradient_large+gated_sum"),
]


@pytest.mark.parametrize("size,kwargs,forward,gradient", FLOATS, ids=lambda x: str(x))
def test_each_kernel_of_floats_by_name(stream, size, kwargs, forward, gradient):  # noqa: F811
    D = owned("float")
    met = check(D, *size, seed=1, **kwargs)
    assert forward is None or met[0] == forward, met
    assert gradient is None or met[1] == gradient, met
    D.free()


@pytest.mark.parametrize("rows,hidden,kernel", [(1300, 2021, "gated_pairs"), (700, 1100, "gated_medium")])
def test_floats_beyond_the_range_of_halves(stream, rows, hidden, kernel):  # noqa: F811
    """Elements of 2^115 times elements of 2^-116: powers of two, whose products and sums are exact."""
    D = owned("float")
    width = 64
    x, weights = np.full((rows, width), 2.0 ** 115, np.float32), np.full((2 * hidden, width), 2.0 ** -116, np.float32)
    inner, pre = D.tensor(np.zeros((rows, hidden))), D.tensor(np.zeros((rows, 2 * hidden)))
    blocks.gated_gemm(inner, pre, D.tensor(x), D.tensor(weights), activation="relu")
    assert capi.last_kernel() == kernel
    assert np.all(read(pre) == 32.0) and np.all(read(inner) == 1024.0)
    D.free()


@pytest.mark.parametrize("grouped", [False, True])
def test_large_elements_that_meet_none(stream, grouped):  # noqa: F811
    """Rows of both operands with one element 2^40 above the others, which meets a zero or an element as far below: what the others come to is
    held to the bar of a float sum.  Rows of zeros, absent rows, and tiles without such rows beside them; in place, too."""
    D = owned("float")
    rng = np.random.default_rng(17)
    rows, width, hidden = 3000, 1000, 2300
    x = rng.standard_normal((rows, width)).astype(np.float32)
    weights = (rng.standard_normal((2 * hidden, width)) / 32).astype(np.float32)
    x[100:1400, 0] *= np.float32(2.0 ** 40)
    weights[:, 0] *= np.where(np.arange(2 * hidden) % 3 == 0, 0, np.float32(2.0 ** -40)).astype(np.float32)
    weights[500:520, 1] *= np.float32(2.0 ** 45)
    x[:, 1] = 0
    x[7], x[1200], weights[3], weights[hidden + 600] = 0, 0, 0, 0
    index = np.arange(rows)
    index[[8, 700, 2999]] = -1, rows, rows + 5
    inner, pre = D.tensor(np.zeros((rows, hidden))), D.tensor(np.zeros((rows, 2 * hidden)))
    if grouped:
        blocks.gated_gemm(inner, pre, D.tensor(x), D.tensor(np.stack([weights, -weights])), D.tensor([0, 1300, rows], "int"), D.tensor(index, "int"),
                          activation="relu")
    else:
        blocks.gated_gemm(inner, pre, D.tensor(x), D.tensor(weights), activation="relu")
    assert capi.last_kernel() == "gated_pairs"
    taken = x.astype(np.float64)
    if grouped:
        taken[[8, 700, 2999]] = 0
        taken[1300:] *= -1
    w = weights.astype(np.float64)
    got = read(pre)
    close(got, taken @ w.T, (width + 4) * D.u * (abs(taken) @ abs(w).T) + 2.0 ** -149, 1.0)
    assert np.array_equal(read(inner), np.maximum(got[:, :hidden], 0) * got[:, hidden:])
    d = rng.standard_normal((rows, width)).astype(np.float32)
    back = rng.standard_normal((width, hidden)).astype(np.float32)
    d[50:900, 3] *= np.float32(2.0 ** 41)
    back[3] = np.where(np.arange(hidden) % 4 == 0, 0, back[3] * np.float32(2.0 ** -41))
    back[11, 40:70] *= np.float32(2.0 ** 44)
    d[:, 11], d[77], back[:, 55] = 0, 0, 0
    ones = D.tensor(np.ones((rows, 2 * hidden)))
    args = (D.tensor(back),) if not grouped else (D.tensor(np.stack([back, back])),)
    blocks.gated_gemm_gradient(ones, None, D.tensor(d), *args, ones, *((D.tensor([0, 1700, rows], "int"),) if grouped else ()), activation="relu")
    assert capi.last_kernel() == "gated_gradient_pairs"
    d, back = d.astype(np.float64), back.astype(np.float64)
    want, bar = d @ back, (width + 4) * D.u * (abs(d) @ abs(back)) + 2.0 ** -149
    got = read(ones)
    close(got[:, :hidden], want, bar, 1.0)
    close(got[:, hidden:], want, bar, 1.0)
    D.free()
