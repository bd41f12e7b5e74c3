"""The kernels that training steps take, at the least sizes that reach them: larger tiles, several tokens or rows to a group of
lanes, operands that the caches do not hold, lists that are added up by a launch of their own.  The kernel that ran is asserted
where its name tells; formulas and bars are those of tests/test_gpu_blocks.py."""
import numpy as np
import pytest

from cortex_amd import blocks
from cortex_amd import capi
from cortex_amd import optimize
from cortex_amd import tensor as ct
from test_gpu_blocks import D, Owned, check_norm, close, grouped64, norm_case, offsets_of, read, stream  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu

PAST_THE_CACHES = 256 << 20     # bytes that the last-level cache holds


# ------------------------------------------------------------------------------------------------- products by group

def check_products(D, size, trans_b, kernel):
    groups, rows, k, n = size
    for turn, (kind, whole, alpha, beta) in enumerate((("any", True, 1.0, 0.0), ("short", False, 1.5, 0.0), ("any", False, -0.5, 0.75))):
        rng = np.random.default_rng(rows + k + turn)
        make = (lambda *s: rng.integers(-7, 8, s).astype(D.type)) if whole else (lambda *s: rng.standard_normal(s).astype(D.type))
        offsets = offsets_of(rng, groups, rows, kind)
        a_rows = rows // 2
        index = rng.integers(0, a_rows, rows)
        index[::7] = rng.choice([-1, a_rows, 1 << 30], len(index[::7]))
        a, c = make(a_rows, k), make(rows, n)
        b = make(groups, n, k) if trans_b else make(groups, k, n)
        tc = D.block(c, turn)
        blocks.grouped_gemm(tc, trans_b, alpha, D.block(a, turn), D.tensor(b), beta, D.tensor(offsets, "int"), index=D.tensor(index, "int"))
        assert capi.last_kernel() == kernel
        want, scale = grouped64(a, index, b, trans_b, offsets, c, alpha, beta)
        got = read(tc)
        inside = np.zeros(rows, bool)
        inside[offsets[0]:offsets[-1]] = True
        assert np.array_equal(got[~inside], c[~inside]), "rows of no group were written"
        if whole:
            assert np.array_equal(got.astype(np.float64), want)
        else:
            close(got, want, scale, (k + 4) * D.u, kind)


def rows64(x, index):
    return np.where(((index >= 0) & (index < len(x)))[:, None], x[np.clip(index, 0, len(x) - 1)], 0).astype(np.float64)


def check_products_over_rows(D, size, kernel):
    groups, rows, m, n = size
    for turn, (kind, whole, alpha, beta) in enumerate((("any", True, 1.0, 0.0), ("short", False, 1.5, 0.0), ("any", False, -0.5, 0.75))):
        rng = np.random.default_rng(rows + m + turn)
        make = (lambda *s: rng.integers(-7, 8, s).astype(D.type)) if whole else (lambda *s: rng.standard_normal(s).astype(D.type))
        offsets = offsets_of(rng, groups, rows, kind)
        a_rows = max(1, rows // 2)
        ia, ib = rng.integers(0, a_rows, rows), rng.integers(0, rows + 3, rows)
        ia[::9], ib[1::11] = -1, rows + 3
        a, b, c = make(a_rows, m), make(rows + 3, n), make(groups, m, n)
        tc = D.tensor(c)
        blocks.grouped_gemm_weights(tc, alpha, D.block(a, turn), D.block(b, 1), beta, D.tensor(offsets, "int"), a_index=D.tensor(ia, "int"),
                                    b_index=D.tensor(ib, "int"))
        assert capi.last_kernel() == kernel
        got = read(tc)
        for e in range(groups):
            i = slice(offsets[e], offsets[e + 1])
            x, y = rows64(a, ia[i]), rows64(b, ib[i])
            want = alpha * (x.T @ y) + beta * c[e].astype(np.float64)
            if whole:
                assert np.array_equal(got[e].astype(np.float64), want), (kind, e)
            else:
                close(got[e], want, abs(alpha) * (np.abs(x).T @ np.abs(y)) + np.abs(beta * c[e]), (len(x) + 4) * D.u, kind)


PRODUCTS = {(12, 65, 32, 996): "grouped_thin", (1, 4933, 33, 68): "grouped_medium", (3, 900, 200, 700): "grouped_medium",
            (3, 76, 1010, 36): "grouped_medium+grouped_sum", (3, 5763, 32, 132): "grouped_large", (2, 3000, 70, 1100): "grouped_large",
            (3, 2000, 300, 1030): "grouped_large", (6, 3140, 2366, 79): "grouped_large+grouped_sum"}


@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("size", PRODUCTS, ids=str)
def test_products_of_each_tile(stream, size, trans_b):
    D = Owned("float")
    D.u, D.type = 2.0 ** -24, np.float32
    check_products(D, size, trans_b, PRODUCTS[size])
    D.free()


# tiles of 32 a side, and of 64: the least of each, uneven groups over several, and sums in parts
PRODUCTS_IN_DOUBLE = {(3, 700, 300, 520): "grouped_double", (12, 414, 37, 1344): "grouped_double", (2, 3000, 70, 1100): "grouped_double",
                      (2, 4000, 100, 1030): "grouped_double", (4, 8156, 3168, 42): "grouped_double+grouped_sum"}


@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("size", PRODUCTS_IN_DOUBLE, ids=str)
def test_products_of_each_tile_in_double(stream, size, trans_b):
    D = Owned("double")
    D.u, D.type = 2.0 ** -53, np.float64
    check_products(D, size, trans_b, PRODUCTS_IN_DOUBLE[size])
    D.free()


PRODUCTS_OVER_ROWS = {(3, 500, 300, 200): "grouped_weights_medium", (1, 402, 37, 34): "grouped_weights_medium+grouped_sum",
                      (12, 73, 662, 69): "grouped_weights_large", (12, 3000, 520, 500): "grouped_weights_large",
                      (1, 4981, 73, 1548): "grouped_weights_large+grouped_sum"}


@pytest.mark.parametrize("size", PRODUCTS_OVER_ROWS, ids=str)
def test_products_over_rows_of_each_tile(stream, size):
    D = Owned("float")
    D.u, D.type = 2.0 ** -24, np.float32
    check_products_over_rows(D, size, PRODUCTS_OVER_ROWS[size])
    D.free()


PRODUCTS_OVER_ROWS_IN_DOUBLE = {(3, 700, 300, 520): "grouped_weights_double", (12, 77, 3808, 34): "grouped_weights_double",
                                (12, 3000, 520, 500): "grouped_weights_double", (1, 5395, 173, 2012): "grouped_weights_double+grouped_sum"}


@pytest.mark.parametrize("size", PRODUCTS_OVER_ROWS_IN_DOUBLE, ids=str)
def test_products_over_rows_of_each_tile_in_double(stream, size):
    D = Owned("double")
    D.u, D.type = 2.0 ** -53, np.float64
    check_products_over_rows(D, size, PRODUCTS_OVER_ROWS_IN_DOUBLE[size])
    D.free()


def test_products_over_rows_of_large_tiles_and_an_operand_beyond_four_gib(stream):
    """Rows that begin past 2^32 bytes, in tiles of 128: whole numbers, every sum exact."""
    D = Owned("float")
    rng = np.random.default_rng(71)
    ld, a_rows = 1 << 16, (1 << 14) + 40
    groups, rows, m, n = 12, 600, 520, 500
    whole = ct.new_tensor([a_rows * ld], datatype="float")
    D.kept.append(whole)
    index = np.concatenate([rng.integers(0, 40, rows // 2), rng.integers(a_rows - 40, a_rows, rows - rows // 2)])[rng.permutation(rows)]
    small = rng.integers(-7, 8, (a_rows, m)).astype(np.float32)
    for r in np.unique(index):
        row = D.tensor(small[r])
        capi.call("ct_memcpy_async", whole.buffer.ptr + 4 * ld * int(r), row.buffer.ptr, 4 * m, capi.COPY_D2D, stream.handle)
    a = ct.Tensor(whole.device, {"shape": [a_rows, m], "strides": [ld, 1]}, whole.buffer)
    b, offsets = rng.integers(-7, 8, (rows, n)).astype(np.float32), offsets_of(rng, groups, rows, "any")
    tc = D.tensor(np.zeros((groups, m, n)))
    blocks.grouped_gemm_weights(tc, 1.0, a, D.tensor(b), 0.0, D.tensor(offsets, "int"), a_index=D.tensor(index, "int"))
    assert capi.last_kernel() == "grouped_weights_large"
    x, got = small[index].astype(np.float64), read(tc)
    for e in range(groups):
        i = slice(offsets[e], offsets[e + 1])
        assert np.array_equal(got[e].astype(np.float64), x[i].T @ b[i])
    D.free()


def same_classes(got, want, scale, bar, what):
    """NaN and infinities where the sum of the products has them; else within the bar.  A sum of finite products that come near the
    largest float may pass it on the way: only its being finite or not is left open."""
    got, sure = got.astype(np.float64), (scale <= 1e38) | ~np.isfinite(scale)
    for cls in (np.isnan, np.isposinf, np.isneginf):
        assert np.array_equal(cls(got)[sure], cls(want)[sure]), what
    fine = sure & np.isfinite(want)
    off = np.abs(got[fine] - want[fine]) - bar[fine]
    assert np.all(off <= 0), (what, off.max())


@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("size", [(1, 4933, 33, 68), (3, 900, 200, 700), (3, 76, 1010, 36), (3, 5763, 32, 132), (6, 3140, 2366, 79)], ids=str)
def test_products_of_what_is_not_finite_in_each_tile(stream, size, trans_b):
    """Infinities, NaN and floats at the ends of their range, in operands whose products are formed in pieces and again from the
    floats; rows of indexes that lie outside are zeros also beside them.  Bar: 1e-5 of the sum of magnitudes, as for gemm!, and half of
    the least float for each of the k products."""
    D = Owned("float")
    groups, rows, k, n = size
    rng = np.random.default_rng(72)
    a, b = rng.standard_normal((rows, k)).astype(np.float32), rng.standard_normal((groups, n, k)).astype(np.float32)
    a[1, 3], a[2, 0], a[3, k - 1], a[5, 4] = np.inf, np.nan, 3e38, -np.inf
    a[4] *= np.float32(1e-38)
    a[rows - 1, 7], a[rows // 2] = np.nan, a[rows // 2] * np.float32(1e20)
    b[0, 5, 2], b[groups - 1, n - 1, k - 1] = -np.inf, np.inf
    b[groups - 1, 0] *= np.float32(1e18)
    index = np.arange(rows)
    index[8::5] = -1
    index[rows - 1] = rows - 1
    offsets = offsets_of(rng, groups, rows, "any")
    tc = D.tensor(np.zeros((rows, n)))
    stored = b if trans_b else np.ascontiguousarray(b.transpose(0, 2, 1))
    blocks.grouped_gemm(tc, trans_b, 1.0, D.tensor(a), D.tensor(stored), 0.0, D.tensor(offsets, "int"), index=D.tensor(index, "int"))
    kernel = capi.last_kernel()
    assert kernel.startswith(("grouped_medium", "grouped_large"))
    with np.errstate(all="ignore"):
        want, scale = grouped64(a, index, b, True, offsets, np.zeros((rows, n), np.float32), 1.0, 0.0)
        assert np.isnan(want).any() and np.isposinf(want).any() and np.isneginf(want).any() and np.isfinite(want).any()
        same_classes(read(tc), want, scale, 1e-5 * scale + k * 2.0 ** -150, kernel)
    D.free()


@pytest.mark.parametrize("size", [(3, 500, 300, 200), (1, 402, 37, 34), (12, 73, 662, 69), (1, 4981, 73, 1548)], ids=str)
def test_products_over_rows_of_what_is_not_finite(stream, size):
    """The same of sums over rows, which indexes name."""
    D = Owned("float")
    groups, rows, m, n = size
    rng = np.random.default_rng(73)
    a, b = rng.standard_normal((rows, m)).astype(np.float32), rng.standard_normal((rows, n)).astype(np.float32)
    a[1, 3], a[2, 0], a[3, m - 1], a[rows - 1, 4] = np.inf, np.nan, 3e38, -np.inf
    a[:, 5] *= np.float32(1e-38)
    a[:, 6] *= np.float32(1e20)
    b[rows // 2, 1], b[7, n - 1] = np.inf, -np.inf
    b[:, 2] *= np.float32(1e18)
    ia, ib = np.arange(rows), rng.permutation(rows)
    ia[10::5], ib[11::6] = -1, rows
    offsets = offsets_of(rng, groups, rows, "any")
    tc = D.tensor(np.zeros((groups, m, n)))
    blocks.grouped_gemm_weights(tc, 1.0, D.tensor(a), D.tensor(b), 0.0, D.tensor(offsets, "int"), a_index=D.tensor(ia, "int"), b_index=D.tensor(ib, "int"))
    kernel, got = capi.last_kernel(), read(tc)
    classes = np.zeros(3, bool)
    with np.errstate(all="ignore"):
        for e in range(groups):
            i = slice(offsets[e], offsets[e + 1])
            x, y = rows64(a, ia[i]), rows64(b, ib[i])
            want, scale = x.T @ y, np.abs(x).T @ np.abs(y)
            classes |= [np.isnan(want).any(), np.isinf(want).any(), np.isfinite(want).any()]
            same_classes(got[e], want, scale, 1e-5 * scale + len(x) * 2.0 ** -150, (kernel, e))
    assert classes.all()
    D.free()


# ------------------------------------------------------------------------------------------------- combining

def check_combine(D, n, k, width, sampled=None):
    """Both directions; where `sampled` is given, that many tokens are compared."""
    rng = np.random.default_rng(n + width)
    slots = rng.permutation(n * k).reshape(n, k)
    slots = np.where(rng.random((n, k)) < 0.1, rng.choice([-1, n * k, 1 << 30], (n, k)), slots)
    rows, weights, dy = (rng.standard_normal(s, np.float32).astype(D.type) for s in ((n * k, width), (n, k), (n, width)))
    tr, tw, ts, tdy = D.block(rows, 1), D.tensor(weights), D.tensor(slots, "int"), D.tensor(dy)
    out, to, dw = D.block(np.zeros((n, width)), 1), D.tensor(np.full((n * k, width), 5.0)), D.tensor(np.full((n, k), 9.0))
    blocks.combine_experts(out, tr, tw, ts)
    blocks.combine_experts_gradient(to, dw, tdy, tr, tw, ts)
    some = np.arange(n) if sampled is None else np.unique(np.concatenate([[0, 1, n - 2, n - 1], rng.integers(0, n, sampled)]))
    have = ((slots >= 0) & (slots < n * k))[some]
    at = np.where(have, slots[some], 0)
    taken = np.where(have[:, :, None], rows[at].astype(np.float64), 0)
    terms = weights[some].astype(np.float64)[:, :, None] * taken
    close(read(out)[some], terms.sum(1), np.abs(terms).sum(1), (k + 4) * D.u, "output")
    dots = taken * dy[some, None, :].astype(np.float64)
    close(read(dw)[some], dots.sum(2), np.abs(dots).sum(2), (width + 4) * D.u, "weights gradient")
    got = read(to)
    assert np.array_equal(got[at[have]], (weights[some][:, :, None] * dy[some][:, None, :])[have]), "rows gradient"
    named = np.zeros(n * k, bool)
    named[slots[(slots >= 0) & (slots < n * k)]] = True
    assert np.all(got[~named] == 5.0), "rows that no slot names were written"


# several tokens to a wave, the last run a short one, of one part and of several; over 1024 assignments of more than 64 pieces
@pytest.mark.parametrize("size", [(20011, 1, 5), (33001, 2, 64), (40009, 3, 70), (9001, 8, 600), (5003, 32, 1040), (700, 2, 1000), (1100, 1, 257),
                                  (1030, 4, 1031)], ids=str)
def test_combine_of_many_tokens(D, size):
    check_combine(D, *size, sampled=3000)


# 16, 64 and 256 lanes to an assignment
@pytest.mark.parametrize("size", [(70001, 8, 119), (30011, 2, 1001), (6007, 4, 2801)], ids=str)
def test_combine_past_the_caches(stream, size):
    n, k, width = size
    assert n * (k + 1) * width * 4 > PAST_THE_CACHES
    D = Owned("float")
    D.u, D.type = 2.0 ** -24, np.float32
    check_combine(D, n, k, width, sampled=2000)
    D.free()


def test_combine_in_double_past_the_caches(stream):
    D = Owned("double")
    D.u, D.type = 2.0 ** -53, np.float64
    check_combine(D, 12007, 3, 801, sampled=2000)
    D.free()


# ------------------------------------------------------------------------------------------------- norms

# more rows than groups of lanes: 16, 64, 256 and 1024 lanes to a row
ROWS_TO_A_GROUP = [(60001, 40), (9001, 300), (2503, 1500), (700, 6001)]


@pytest.mark.parametrize("kinds", [("rms", "rms"), ("layer", "layer"), ("none", "layer")], ids="-".join)
@pytest.mark.parametrize("shape", ROWS_TO_A_GROUP, ids=str)
def test_norms_of_several_rows_to_a_group(D, shape, kinds):
    check_norm(D, *shape, *kinds, "row" if kinds[0] == "rms" else "column", biases=kinds[0] == "layer", residual=True, pad=1, seed=7)


def check_norm_in_place(D, rows, width, post, pre, gate):
    """The results in place of the operands, each pair that may be, and the gradients: the same bits as into memory of their own."""
    rng = np.random.default_rng(74)
    z, r, p = norm_case(rng, D, rows, width, post, pre, gate, post == "layer")
    tp = {k: D.tensor(v) for k, v in p.items()}
    d = blocks.norm_descriptor(post=post, pre=pre, residual_scale=0.75)
    mine, zeros = [], np.zeros((rows, width))
    keep = lambda x: mine.append(D.tensor(x)) or mine[-1]
    tz, tr, out, h, stats = keep(z), keep(r), keep(zeros), keep(zeros), keep(np.zeros((4, rows)))
    blocks.norm_residual(out, h, stats, tz, tr, tp, d)
    want = [read(out), read(h), read(stats)]
    for over_out, over_h in (("z", "r"), ("r", "z"), (None, "r"), (None, "z"), ("r", None), ("z", None)):
        at = {"z": keep(z), "r": keep(r), None: keep(zeros)}
        stats2 = keep(np.zeros((4, rows)))
        blocks.norm_residual(at[over_out], at[over_h], stats2, at["z"], at["r"], tp, d)
        for a, b in zip(want, (at[over_out], at[over_h], stats2)):
            assert np.array_equal(a, read(b)), (over_out, over_h)
    dout, dh = rng.standard_normal((rows, width)), rng.standard_normal((rows, width))
    results = []
    for over_dz, over_dr in ((None, None), ("out", "h"), ("h", "out"), ("h", None), (None, "out")):
        at = {"out": keep(dout), "h": keep(dh)}
        dz, dr = at.get(over_dz) or keep(zeros), at.get(over_dr) or keep(zeros)
        g = {k: keep(np.full(v.shape, 3.0)) for k, v in p.items()}
        blocks.norm_residual_gradient(dz, dr, g, at["out"], at["h"], tz, out, stats, tp, d)
        results.append([read(t) for t in (dz, dr, *g.values())])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert np.array_equal(a, b) and np.any(a != 0)


@pytest.mark.parametrize("kinds", [("rms", "layer"), ("layer", "rms"), ("none", "rms")], ids="-".join)
@pytest.mark.parametrize("shape", [(5, 3), (40, 70), (30, 1003), (9, 4100), (4, 16385)] + ROWS_TO_A_GROUP, ids=str)
def test_norms_in_place(D, shape, kinds):
    check_norm_in_place(D, *shape, *kinds, "column" if kinds[0] == "rms" else "row")


# operands that the last-level cache does not hold: 16, 64, 256 and 1024 lanes to a row, all off the 16-byte grid
@pytest.mark.parametrize("shape", [(242003, 70), (16901, 1001), (8209, 2049), (1697, 10001)], ids=str)
def test_norms_past_the_caches(stream, shape):
    rows, width = shape
    assert 4 * rows * width * 4 > PAST_THE_CACHES
    D = Owned("float")
    D.u, D.type = 2.0 ** -24, np.float32
    check_norm(D, *shape, "layer" if width > 1500 else "rms", "layer" if width < 1500 else "rms", "column", biases=True, residual=True, pad=1, seed=8)
    D.free()


@pytest.mark.parametrize("shape", [(130003, 65), (1800, 5001)], ids=str)
def test_norms_in_double_past_the_caches(stream, shape):
    D = Owned("double")
    D.u, D.type = 2.0 ** -53, np.float64
    check_norm(D, *shape, "layer", "rms", "row", biases=True, residual=True, pad=0, seed=9)
    D.free()


def test_norm_gradients_in_place_past_the_caches(stream):
    D = Owned("float")
    D.u, D.type = 2.0 ** -24, np.float32
    check_norm_in_place(D, 45007, 301, "rms", "rms", "full")
    D.free()


# ------------------------------------------------------------------------------------------------- clipping

def check_clip(D, stream, sizes, seed):
    rng = np.random.default_rng(seed)
    n = sum(sizes)
    host = (rng.standard_normal(n, np.float32) * np.repeat(10.0 ** rng.uniform(-3, 1, len(sizes)), sizes)).astype(D.type)
    ends = np.cumsum([0] + list(sizes))
    norm64 = np.sqrt((host.astype(np.float64) ** 2).sum())
    bar = 4 * D.u + n * 2.0 ** -53
    flat, into, result = D.tensor(host), D.tensor(np.full(n + 1, 7.25)), D.tensor(np.zeros(2))
    gradients = [flat.buffer.sub_buffer(int(at), int(s)) for at, s in zip(ends, sizes)]
    outputs = [into.buffer.sub_buffer(int(at) + 1, int(s)) for at, s in zip(ends, sizes)]
    backend = optimize.Backend(stream, D.datatype)
    for limit, in_place in ((norm64 / 3, False), (norm64 * 2, False), (norm64 / 5, True)):
        optimize.clip_gradients(backend, gradients, limit, result, None if in_place else outputs)
        norm, factor = read(result)
        want = min(1.0, limit / norm64)
        assert abs(float(norm) - norm64) <= bar * norm64 and abs(float(factor) - want) <= bar * want
        assert np.array_equal(read(flat if in_place else into)[0 if in_place else 1:], host * factor)
        assert in_place or read(into)[0] == 7.25


def test_clip_gradients_of_many_sums(D, stream):
    """Four tables of tensors and 2400 sums: a launch of its own adds them, and the factor is read back."""
    size = 4096 // np.dtype(D.type).itemsize
    check_clip(D, stream, [5 * size + 1] * 400, 75)


def test_clip_gradients_past_the_caches(stream):
    """Over 256 MiB of gradients and results, three tables, every launch full and its blocks at several pieces each."""
    D = Owned("float")
    D.u, D.type = 2.0 ** -24, np.float32
    sizes = [9_000_001, 16, 14_000_003, 1] + [100_003] * 296
    assert 2 * 4 * sum(sizes) > PAST_THE_CACHES
    check_clip(D, stream, sizes, 76)
    D.free()
