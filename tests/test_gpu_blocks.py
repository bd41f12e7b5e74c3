"""The operators of residual blocks with experts against their formulas in 64 bits (numpy), at sizes, strides and masks
where they can go wrong.

Bars, fixed ahead: with u = 2^-24 (float) or 2^-53 (double), a value that is formed by few roundings after sums in trees is
held to 64 u of the sum of the magnitudes of its terms; a sum of k products taken one after the other to (k + 4) u of that;
whole numbers whose sums stay below 2^24 exactly; indexes exactly.
"""
import itertools

import numpy as np
import pytest

from cortex_amd import blocks
from cortex_amd import capi
from cortex_amd import driver as drv
from cortex_amd import optimize
from cortex_amd import tensor as ct

pytestmark = pytest.mark.gpu

NUMPY = {"float": np.float32, "double": np.float64}
UNIT = {"float": 2.0 ** -24, "double": 2.0 ** -53}


@pytest.fixture()
def stream():
    capi.call("ct_set_device", 0)
    capi.call("ct_set_debug_sync", 1)
    s = drv.HipDriver().default_device().create_stream()
    with ct.tensor_context(s, "float"):
        yield s
    s.release()


@pytest.fixture()
def as_released():
    """Debug-sync mode off, as a user runs, and on again for the other tests."""
    capi.call("ct_set_device", 0)
    capi.call("ct_set_debug_sync", 0)
    yield
    capi.call("ct_set_debug_sync", 1)


class Owned:
    """Tensors on the device, freed together; a matrix may be a block of a wider one, whose rest must stay as it is."""

    def __init__(self, datatype):
        self.datatype, self.kept = datatype, []

    def tensor(self, data, datatype=None):
        data = np.asarray(data)
        t = ct.to_tensor(data if data.size else np.zeros(1), datatype or self.datatype)
        if not data.size:
            t = ct.Tensor(t.device, {"shape": list(data.shape), "strides": strides_of(data.shape)}, t.buffer)
        self.kept.append(t)
        return t

    def block(self, data, pad):
        """A matrix whose rows lie `pad` further apart than they are long, behind one element of the buffer."""
        data = np.asarray(data, NUMPY[self.datatype])
        whole = np.full((data.shape[0], data.shape[1] + pad), 7.25, data.dtype)
        whole[:, :data.shape[1]] = data
        whole = np.concatenate([np.full(1, 7.25, data.dtype), whole.reshape(-1)])
        t = self.tensor(whole)
        view = ct.Tensor(t.device, {"shape": list(data.shape), "strides": [data.shape[1] + pad, 1]},
                         t.buffer.sub_buffer(1, whole.size - 1))
        view.whole = t
        return view

    def free(self):
        for t in self.kept:
            t.buffer.release()


def strides_of(shape):
    out, m = [], 1
    for n in reversed(shape):
        out.insert(0, m)
        m *= max(n, 1)
    return out


def read(t):
    if hasattr(t, "whole"):
        flat = ct.to_array_of_type(t.whole, t.get_datatype())
        rows, columns = t.shape()
        whole = flat[1:].reshape(rows, -1)
        assert flat[0] == 7.25 and np.all(whole[:, columns:] == 7.25), "written beside the rows"
        return whole[:, :columns].copy()
    return ct.to_array_of_type(t, t.get_datatype()).reshape(t.shape())


@pytest.fixture(params=["float", "double"])
def D(request, stream):
    owned = Owned(request.param)
    owned.u = UNIT[request.param]
    owned.type = NUMPY[request.param]
    yield owned
    owned.free()


def close(got, want, scale, bar, what=""):
    got, want, scale = (np.asarray(x, np.float64) for x in (got, want, scale))
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.all(np.isfinite(got)), what
    off = np.abs(got - want) - bar * scale
    assert np.all(off <= 0), f"{what}: {np.max(np.abs(got - want) / np.maximum(scale, 1e-300)) / bar:.3g} times the bar"


# ------------------------------------------------------------------------------------------------- norms

def norm64(x, kind, scale, bias, eps):
    if kind == "none":
        return x, x, np.ones((len(x), 1))
    c = x - x.mean(1, keepdims=True) if kind == "layer" else x
    rate = 1 / np.sqrt((c * c).mean(1, keepdims=True) + eps)
    hat = c * rate
    return hat * (1 if scale is None else scale) + (0 if bias is None else bias), hat, rate


def norm_t64(y, hat, rate, kind):
    if kind == "none":
        return y
    return rate * (y - (y.mean(1, keepdims=True) if kind == "layer" else 0) - hat * (y * hat).mean(1, keepdims=True))


def block64(z, r, p, post, pre, c, eps):
    u, zh, zr = norm64(z, post, p.get("post-scale"), p.get("post-bias"), eps)
    out = p.get("gate", 1.0) * u + (0 if r is None else c * r)
    h, oh, orate = norm64(out, pre, p.get("pre-scale"), p.get("pre-bias"), eps)
    return out, h, (u, zh, zr, oh, orate)


def gradient64(dout, dh, z, r, p, post, pre, c, eps):
    """Gradients by the formulas, and the magnitudes of what they are summed of."""
    out, h, (u, zh, zr, oh, orate) = block64(z, r, p, post, pre, c, eps)
    d, g = dout.copy(), {}
    if pre != "none":
        d = d + norm_t64(dh * p.get("pre-scale", 1.0), oh, orate, pre)
        g["pre-scale"], g["pre-bias"] = dh * oh, dh
    gate = p.get("gate", np.ones((1, 1)))
    du = d * gate
    g["gate"] = d * u
    if post != "none":
        g["post-scale"], g["post-bias"] = du * zh, du
    dz = norm_t64(du * p.get("post-scale", 1.0), zh, zr, post) if post != "none" else du

    def summed(name, x):
        if name == "gate":
            axes = tuple(i for i in (0, 1) if p["gate"].shape[i] == 1)
            return x.sum(axis=axes, keepdims=True) if axes else x
        return x.sum(0)
    return dz, c * d, {k: summed(k, v) for k, v in g.items() if k in p}, {k: summed(k, np.abs(v)) for k, v in g.items() if k in p}


KINDS = [("rms", "rms"), ("layer", "layer"), ("none", "rms"), ("layer", "none"), ("none", "none"), ("rms", "layer")]
# rows held by 16, 64, 256 and 1024 lanes, at their edges and off the 16-byte grid, and rows that no block holds
SHAPES = [(1, 1), (3, 2), (5, 16), (33, 63), (7, 129), (40, 257), (9, 1000), (3, 1025), (6, 2049), (2, 4097), (700, 70)]
LONG = [(2, 16385), (3, 20001)]


def norm_case(rng, D, rows, width, post, pre, gate, biases, residual=True):
    make = lambda *s, mean=0.0, std=1.0: (mean + std * rng.standard_normal(s)).astype(D.type)
    z, r = make(rows, width, mean=0.3), make(rows, width, std=2.0) if residual else None
    p = {}
    for place, kind in (("post", post), ("pre", pre)):
        if kind != "none":
            p[place + "-scale"] = make(width, mean=1.0, std=0.2)
            if biases:
                p[place + "-bias"] = make(width, std=0.3)
    if gate:
        p["gate"] = make(*{"scalar": (1, 1), "column": (1, width), "row": (rows, 1), "full": (rows, width)}[gate], mean=0.5)
    return z, r, p


def check_norm(D, rows, width, post, pre, gate, biases, residual, pad, seed, eps=1e-5, c=0.75):
    rng = np.random.default_rng(seed)
    z, r, p = norm_case(rng, D, rows, width, post, pre, gate, biases, residual)
    f = lambda x: None if x is None else x.astype(np.float64)
    z64, r64, p64 = f(z), f(r), {k: f(v) for k, v in p.items()}
    eps64 = float(D.type(eps))
    tz, tr = D.block(z, pad), D.block(r, pad + 1) if residual else None
    tp = {k: D.tensor(v) for k, v in p.items()}
    out = D.block(np.zeros((rows, width)), pad)
    h = D.block(np.zeros((rows, width)), pad + 2) if pre != "none" else None
    stats = D.tensor(np.zeros((4, rows)))
    d = blocks.norm_descriptor(post=post, pre=pre, epsilon=eps, residual_scale=c)
    blocks.norm_residual(out, h, stats, tz, tr, tp, d)
    out64, h64, (u, zh, zr, oh, orate) = block64(z64, r64, p64, post, pre, c, eps64)
    # a value's terms; a whole row's are in its statistics
    spread = lambda x: np.abs(x) + np.abs(x).max(1, keepdims=True)
    out_scale = spread(np.abs(p64.get("gate", 1.0)) * (np.abs(u) + np.abs(p64.get("post-bias", 0.0)) + np.abs(zr * z64) * np.abs(p64.get("post-scale", 1.0))) + (0 if r is None else c * np.abs(r64)))
    close(read(out), out64, out_scale, 64 * D.u, "output")
    if pre != "none":
        h_scale = spread(orate * out_scale * np.abs(p64.get("pre-scale", 1.0)) + np.abs(p64.get("pre-bias", 0.0)))
        close(read(h), h64, h_scale, 64 * D.u, "normalized")
    # the gradient, from what the call stored
    dout, dh = (rng.standard_normal((rows, width)).astype(D.type) for _ in range(2))
    tdo, tdh = D.block(dout, pad), D.block(dh, pad + 3)
    dz, dr = D.block(np.zeros((rows, width)), pad + 1), D.block(np.zeros((rows, width)), pad)
    tg = {k: D.tensor(np.full(v.shape, 3.0)) for k, v in p.items()}
    blocks.norm_residual_gradient(dz, dr, tg, tdo, tdh if pre != "none" else None, tz, out, stats, tp, d)
    dz64, dr64, g64, g_scale = gradient64(f(dout), f(dh), z64, r64, p64, post, pre, c, eps64)
    # a gradient has the error of the forward's values, whose scale relative to the value is out_scale * orate
    grow = 1 + (orate * out_scale if pre != "none" else 0) + zr * np.abs(z64).max(1, keepdims=True)
    grow = grow.max()
    dr_scale = spread(np.abs(dr64)) + spread(c * (np.abs(f(dout)) + orate * np.abs(f(dh)) * np.abs(p64.get("pre-scale", 1.0))))
    close(read(dr), dr64, dr_scale * grow, 64 * D.u, "residual gradient")
    dz_scale = spread(np.abs(dz64)) + spread(zr * np.abs(p64.get("gate", 1.0)) * np.abs(p64.get("post-scale", 1.0)) * dr_scale / c)
    close(read(dz), dz64, dz_scale * grow, 64 * D.u, "input gradient")
    for k in p:
        full = {"gate": dr_scale / c * (np.abs(u) + 1), "post-scale": np.abs(p64.get("gate", 1.0)) * dr_scale / c * (np.abs(zh) + 1),
                "post-bias": np.abs(p64.get("gate", 1.0)) * dr_scale / c, "pre-scale": np.abs(f(dh)) * (np.abs(oh) + 1), "pre-bias": np.abs(f(dh))}[k]
        if k == "gate":
            axes = tuple(i for i in (0, 1) if p["gate"].shape[i] == 1)
            scale = (full * np.ones((rows, width))).sum(axis=axes, keepdims=True) if axes else full * np.ones((rows, width))
        else:
            scale = (full * np.ones((rows, width))).sum(0)
        close(read(tg[k]), g64[k], scale * grow, 64 * D.u, f"gradient of {k}")


@pytest.mark.parametrize("kinds", KINDS, ids="-".join)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_norm_residual(D, shape, kinds):
    gates = ["column", "row", "full", "scalar", None]
    i = SHAPES.index(shape) + KINDS.index(kinds)
    for n, gate in enumerate((gates[i % 5], gates[(i + 2) % 5])):
        check_norm(D, *shape, *kinds, gate, biases=(i + n) % 2 == 0, residual=(i + n) % 3 != 0, pad=i % 3, seed=i)


@pytest.mark.parametrize("kinds", [("rms", "rms"), ("layer", "layer")], ids="-".join)
@pytest.mark.parametrize("shape", [(37, 70), (37, 95), (300, 150), (13, 191), (9, 300), (9, 383), (200, 700), (7, 767), (5, 1100), (5, 1535), (40, 2500),
                                   (3, 4500), (3, 6143), (4, 9001)], ids=str)
def test_norm_residual_of_three_pieces_to_a_lane(D, shape, kinds):
    """Rows between two and four pieces of 16 bytes to each of the lanes that hold them."""
    check_norm(D, *shape, *kinds, "column", kinds[0] == "layer", True, 1, sum(shape))


@pytest.mark.parametrize("gate", ["column", "row", "full", "scalar", None])
@pytest.mark.parametrize("shape", [(2100, 40), (1111, 300), (600, 1500)], ids=str)
def test_norm_residual_sums_over_many_rows(D, shape, gate):
    check_norm(D, *shape, "layer", "rms", gate, biases=True, residual=True, pad=0, seed=3)
    check_norm(D, *shape, "rms", "rms", gate, biases=False, residual=True, pad=1, seed=4)


@pytest.mark.parametrize("gate", ["column", "row", "full", "scalar", None])
@pytest.mark.parametrize("shape", [(40, 4500), (7, 8192), (300, 9001), (5, 16384)], ids=str)
def test_norm_residual_whose_sums_take_two_passes(D, shape, gate):
    """The sums of scales and of biases, which LDS does not hold together."""
    check_norm(D, *shape, "layer", "layer", gate, biases=True, residual=True, pad=1, seed=6)


def test_norm_gradient_in_place_of_two_passes(D):
    """The gradients of the results overwritten: the same bits as into memory of their own."""
    rng = np.random.default_rng(49)
    rows, width = 30, 8192 if D.datatype == "double" else 12000
    make = lambda *s: rng.standard_normal(s)
    d = blocks.norm_descriptor(post="layer", pre="layer")
    p = {k: D.tensor(make(width)) for k in ("post-scale", "post-bias", "pre-scale", "pre-bias")}
    z, out, h, statistics = D.tensor(make(rows, width)), D.tensor(np.zeros((rows, width))), D.tensor(np.zeros((rows, width))), D.tensor(np.zeros((4, rows)))
    blocks.norm_residual(out, h, statistics, z, D.tensor(make(rows, width)), p, d)
    dout, dh = make(rows, width), make(rows, width)
    results = []
    for in_place in (False, True):
        tout, th = D.tensor(dout), D.tensor(dh)
        dz, dr = (th, tout) if in_place else (D.tensor(np.zeros((rows, width))), D.tensor(np.zeros((rows, width))))
        g = {k: D.tensor(np.zeros(width)) for k in p}
        blocks.norm_residual_gradient(dz, dr, g, tout, th, z, out, statistics, p, d)
        results.append([read(t) for t in (dz, dr, *g.values())])
    for a, b in zip(*results):
        assert np.array_equal(a, b) and np.any(a != 0)


@pytest.mark.parametrize("kinds", [("rms", "rms"), ("layer", "layer"), ("none", "layer")], ids="-".join)
@pytest.mark.parametrize("shape", LONG, ids=str)
def test_norm_residual_of_long_rows(D, shape, kinds):
    for gate in ("column", "row", "full", "scalar"):
        check_norm(D, *shape, *kinds, gate, biases=True, residual=gate != "row", pad=1, seed=5)


def test_norm_residual_in_place(D):
    rng = np.random.default_rng(8)
    for rows, width in ((5, 100), (3, 3000), (2, 17000)):
        z, r, p = norm_case(rng, D, rows, width, "rms", "layer", "column", True)
        tp = {k: D.tensor(v) for k, v in p.items()}
        d = blocks.norm_descriptor(post="rms", pre="layer")
        apart = [D.tensor(x) for x in (np.zeros((rows, width)), np.zeros((rows, width)), np.zeros((4, rows)), z, r)]
        blocks.norm_residual(*apart, tp, d)
        tz, tr, stats = D.tensor(z), D.tensor(r), D.tensor(np.zeros((4, rows)))
        blocks.norm_residual(tr, tz, stats, tz, tr, tp, d)
        for a, b in zip(apart, (tr, tz, stats)):
            assert np.array_equal(read(a), read(b))
        g = [D.tensor(rng.standard_normal((rows, width))) for _ in range(2)]
        to = [D.tensor(np.zeros((rows, width))) for _ in range(2)]
        blocks.norm_residual_gradient(*to, {}, *g, apart[3], apart[0], apart[2], tp, d)
        blocks.norm_residual_gradient(*g, {}, *g, apart[3], apart[0], apart[2], tp, d)
        for a, b in zip(to, g):
            assert np.array_equal(read(a), read(b))


def test_norm_residual_without_what_may_be_absent(D):
    """No statistics, no incoming gradients, no rows."""
    rng = np.random.default_rng(9)
    z, r, p = norm_case(rng, D, 6, 50, "rms", "rms", "row", False)
    tp = {k: D.tensor(v) for k, v in p.items()}
    d = blocks.norm_descriptor(post="rms", pre="rms")
    tz, tr = D.tensor(z), D.tensor(r)
    out, h, out2, h2, stats = (D.tensor(np.zeros(s)) for s in ((6, 50), (6, 50), (6, 50), (6, 50), (4, 6)))
    blocks.norm_residual(out, h, None, tz, tr, tp, d)
    blocks.norm_residual(out2, h2, stats, tz, tr, tp, d)
    assert np.array_equal(read(out), read(out2)) and np.array_equal(read(h), read(h2))
    g = D.tensor(rng.standard_normal((6, 50)))
    for given in ((g, None), (None, g), (None, None)):
        to = [D.tensor(np.full((6, 50), 2.0)) for _ in range(2)]
        tg = {k: D.tensor(np.full(v.shape, 3.0)) for k, v in p.items()}
        blocks.norm_residual_gradient(*to, tg, *given, tz, out, stats, tp, d)
        zero = D.tensor(np.zeros((6, 50)))
        full = [D.tensor(np.full((6, 50), 2.0)) for _ in range(2)]
        tg2 = {k: D.tensor(np.full(v.shape, 3.0)) for k, v in p.items()}
        blocks.norm_residual_gradient(*full, tg2, *(zero if x is None else x for x in given), tz, out, stats, tp, d)
        for a, b in zip(to + list(tg.values()), full + list(tg2.values())):
            assert np.array_equal(read(a), read(b))
    empty = [D.tensor(np.zeros((0, 50))) for _ in range(4)]
    tg = {k: D.tensor(np.full(v.shape, 3.0)) for k, v in p.items() if k != "gate"}
    tp = {k: v for k, v in tp.items() if k != "gate"}
    blocks.norm_residual(empty[0], empty[1], None, empty[2], empty[3], tp, d)
    blocks.norm_residual_gradient(empty[0], empty[1], tg, empty[2], empty[3], empty[0], empty[1], None, tp, d)
    for t in tg.values():
        assert np.all(read(t) == 0)


@pytest.mark.parametrize("kinds", [("rms", "rms"), ("layer", "layer"), ("none", "layer")], ids="-".join)
def test_norm_residual_gradient_is_the_difference(stream, kinds):
    """In double: the directional derivative by central differences of step 1e-5, whose own error is some 1e-10 of the
    second and third derivatives; bar 1e-6."""
    D = Owned("double")
    rng = np.random.default_rng(11)
    rows, width = 9, 37
    z, r, p = norm_case(rng, type("T", (), {"type": np.float64}), rows, width, *kinds, "row", True)
    d = blocks.norm_descriptor(post=kinds[0], pre=kinds[1], residual_scale=0.7)
    dout, dh = rng.standard_normal((rows, width)), rng.standard_normal((rows, width))
    keys = sorted(p)
    direction = {"z": rng.standard_normal(z.shape), "r": rng.standard_normal(r.shape), **{k: rng.standard_normal(p[k].shape) for k in keys}}

    def value(step):
        out, h, stats = D.tensor(np.zeros((rows, width))), D.tensor(np.zeros((rows, width))), D.tensor(np.zeros((4, rows)))
        tz, tr = D.tensor(z + step * direction["z"]), D.tensor(r + step * direction["r"])
        tp = {k: D.tensor(p[k] + step * direction[k]) for k in keys}
        blocks.norm_residual(out, h, stats, tz, tr, tp, d)
        return (read(out) * dout).sum() + (read(h) * dh).sum(), (tz, out, stats, tp)

    _, (tz, out, stats, tp) = value(0.0)
    dz, dr = D.tensor(np.zeros((rows, width))), D.tensor(np.zeros((rows, width)))
    tg = {k: D.tensor(np.zeros(p[k].shape)) for k in keys}
    blocks.norm_residual_gradient(dz, dr, tg, D.tensor(dout), D.tensor(dh), tz, out, stats, tp, d)
    along = (read(dz) * direction["z"]).sum() + (read(dr) * direction["r"]).sum() + sum((read(tg[k]) * direction[k]).sum() for k in keys)
    difference = (value(1e-5)[0] - value(-1e-5)[0]) / 2e-5
    assert abs(along - difference) <= 1e-6 * max(1.0, abs(along))
    D.free()


def test_norm_of_rows_that_are_not_finite(D):
    """An infinity or a NaN stays in its row; a row of zeros is zero over the root of epsilon."""
    rng = np.random.default_rng(12)
    z = rng.standard_normal((5, 200)).astype(D.type)
    z[1, 3], z[2, 7], z[3] = np.inf, np.nan, 0
    tz, out, h = D.tensor(z), D.tensor(np.zeros((5, 200))), D.tensor(np.zeros((5, 200)))
    blocks.norm_residual(out, h, None, tz, None, {}, blocks.norm_descriptor(post="rms", pre="rms"))
    got = read(h)
    assert np.all(np.isfinite(got[[0, 3, 4]])) and np.all(got[3] == 0)
    assert np.isnan(got[1, 3]) and np.all(np.isnan(got[2]))


# ------------------------------------------------------------------------------------------------- routing

def route64(logits, k, renormalize):
    n, e = logits.shape
    x = logits.astype(np.float64)
    order = np.argsort(np.where(np.isnan(x), -np.inf, -x), axis=1, kind="stable")[:, :k]
    values = np.take_along_axis(x, order, 1)
    experts = np.where(np.isneginf(values), -1, order)
    with np.errstate(all="ignore"):
        powers = np.exp(values - values[:, :1])
        total = np.where(experts >= 0, powers, 0).sum(1, keepdims=True) if renormalize else np.exp(x - values[:, :1]).sum(1, keepdims=True)
        weights = np.where(experts >= 0, powers / total, 0.0)
    flat = experts.reshape(-1)
    groups = [np.flatnonzero(flat == i) for i in range(e)]
    placed = np.concatenate(groups)
    tokens, slots = np.full(n * k, -1), np.full(n * k, -1)
    tokens[:len(placed)] = placed // k
    slots[placed] = np.arange(len(placed))
    return experts, weights, np.cumsum([0] + [len(g) for g in groups]), tokens, slots.reshape(n, k)


def run_route(D, logits, k, renormalize, pad=0):
    n, e = logits.shape
    t = D.block(logits, pad) if pad else D.tensor(logits)
    experts, slots = (D.tensor(np.full((n, k), 77), "int") for _ in range(2))
    offsets, tokens = D.tensor(np.full(e + 1, 77), "int"), D.tensor(np.full(n * k, 77), "int")
    weights = D.tensor(np.full((n, k), 7.0))
    blocks.route_experts(experts, weights, offsets, tokens, slots, t, renormalize=renormalize)
    return t, (experts, weights, offsets, tokens, slots)


ROUTES = [(1, 1, 1), (1, 2, 2), (3, 7, 3), (16, 64, 8), (63, 16, 1), (64, 17, 4), (65, 33, 2), (200, 128, 8), (1000, 129, 6),
          (700, 256, 32), (130, 300, 5), (90, 1000, 32), (257, 1024, 3), (5000, 8, 2), (9001, 60, 4),
          (20, 300, 2), (32, 512, 2), (16, 200, 8), (60, 250, 4), (33, 257, 1), (31, 700, 2), (300, 400, 5), (1024, 130, 3), (1025, 500, 3), (8193, 513, 2)]


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("size", ROUTES, ids=str)
def test_route_experts(D, size, renormalize):
    n, e, k = size
    rng = np.random.default_rng(n + e)
    for variant in ("plain", "ties", "closed"):
        logits = rng.standard_normal((n, e)).astype(D.type)
        if variant == "ties":
            logits = np.round(logits * 2) / 2
            logits[logits == 0] = rng.choice([0.0, -0.0], (logits == 0).sum())
        if variant == "closed":
            logits[rng.random((n, e)) < 0.5] = -np.inf
            logits[:: 5] = -np.inf
            logits[1:: 7, :1] = np.finfo(D.type).min    # the type's lowest value is open
        t, got = run_route(D, logits, k, renormalize, pad=n % 3)
        want = route64(logits, k, renormalize)
        for i, what in ((0, "experts"), (2, "offsets"), (3, "tokens"), (4, "slots")):
            assert np.array_equal(read(got[i]), want[i]), (variant, what)
        close(read(got[1]), want[1], want[1], 64 * D.u, f"{variant}: weights")
        # gradient
        dw = rng.standard_normal((n, k)).astype(D.type)
        to = D.block(np.zeros((n, e)), 1)
        blocks.route_experts_gradient(to, D.tensor(dw), got[1], got[0], None if renormalize and n % 2 else t, renormalize=renormalize)
        w, dw64 = want[1], np.where(want[0] >= 0, dw.astype(np.float64), 0)
        common = (w * dw64).sum(1, keepdims=True)
        magnitude = (w * np.abs(dw64)).sum(1, keepdims=True)
        p, spread = np.zeros((n, e)), np.zeros((n, e))
        if not renormalize:
            x = logits.astype(np.float64)
            top = x.max(1, keepdims=True)
            with np.errstate(all="ignore"):
                p = np.where(np.isneginf(top), 0.0, np.exp(x - top) / np.exp(x - top).sum(1, keepdims=True))
        else:
            at = np.where(want[0] >= 0, want[0], 0)
            np.add.at(p, (np.arange(n)[:, None], at), np.where(want[0] >= 0, w, 0))
        np.add.at(spread, (np.arange(n)[:, None], np.where(want[0] >= 0, want[0], 0)), dw64)
        close(read(to), p * (spread - common), p * (np.abs(spread) + magnitude), 64 * D.u, f"{variant}: logits gradient")


def test_route_of_logits_that_are_not_finite(D):
    """NaN is chosen first and makes its row's weights NaN; other rows stay."""
    logits = np.array([[0.0, 1.0, 2.0, 3.0], [0.0, np.nan, 5.0, 1.0], [1.0, np.inf, 0.0, -np.inf], [-np.inf] * 4], D.type)
    _, (experts, weights, offsets, tokens, slots) = run_route(D, logits, 2, True)
    assert read(experts).tolist() == [[3, 2], [1, 2], [1, 0], [-1, -1]]
    w = read(weights)
    assert np.all(np.isfinite(w[[0, 3]])) and np.all(np.isnan(w[1])) and np.isnan(w[2, 0]) and np.all(w[3] == 0)
    assert read(offsets).tolist() == [0, 1, 3, 5, 6] and read(tokens).tolist() == [2, 1, 2, 0, 1, 0, -1, -1]


def test_route_of_no_tokens(D):
    e = 5
    offsets = D.tensor(np.full(e + 1, 9), "int")
    none = lambda *s, **k: D.tensor(np.zeros(s), **k)
    blocks.route_experts(none(0, 2, datatype="int"), none(0, 2), offsets, none(0, datatype="int"), none(0, 2, datatype="int"), none(0, e))
    assert read(offsets).tolist() == [0] * (e + 1)


def test_route_gradient_is_the_difference(stream):
    """In double, step 1e-5, where the choice does not change; bar 1e-7 of magnitudes near one."""
    D = Owned("double")
    rng = np.random.default_rng(21)
    n, e, k = 7, 20, 4
    logits = rng.permuted(np.arange(e) * 0.3, axis=None) + np.zeros((n, 1))
    logits = rng.permuted(logits, axis=1)
    dw, direction = rng.standard_normal((n, k)), rng.standard_normal((n, e))
    for renormalize in (True, False):
        t, got = run_route(D, logits, k, renormalize)
        to = D.tensor(np.zeros((n, e)))
        blocks.route_experts_gradient(to, D.tensor(dw), got[1], got[0], t, renormalize=renormalize)
        value = lambda s: (read(run_route(D, logits + s * direction, k, renormalize)[1][1]) * dw).sum()
        difference = (value(1e-5) - value(-1e-5)) / 2e-5
        assert abs((read(to) * direction).sum() - difference) <= 1e-7
    D.free()


# ------------------------------------------------------------------------------------------------- grouped products

def offsets_of(rng, groups, rows, kind):
    if kind == "one":          # all rows in one group
        cuts = np.sort(rng.choice([0, rows], max(groups - 1, 0)))
    elif kind == "short":      # some rows belong to none
        cuts = np.sort(rng.integers(0, rows + 1, groups + 1))
        return cuts
    else:
        cuts = np.sort(rng.integers(0, rows + 1, max(groups - 1, 0)))
    return np.concatenate([[0], cuts, [rows]]) if groups else np.array([0])


# (groups, rows, k, n): single rows, tiles and their edges, short and long sums, many groups
GROUPED = [(1, 1, 1, 1), (2, 3, 5, 2), (3, 1, 64, 33), (4, 17, 31, 65), (5, 130, 100, 63), (70, 200, 40, 50), (3, 300, 33, 200), (130, 64, 20, 10),
           (2, 700, 257, 130), (8, 1000, 130, 300), (3, 90, 1100, 70), (4, 40, 2050, 300), (2, 2500, 70, 520), (16, 16, 512, 640)]


def grouped64(a, index, b, trans_b, offsets, c, alpha, beta):
    out, scale = c.astype(np.float64).copy(), np.abs(beta * c.astype(np.float64))
    for e in range(len(b)):
        for_rows = slice(offsets[e], offsets[e + 1])
        i = index[for_rows]
        x = np.where(((i >= 0) & (i < len(a)))[:, None], a[np.clip(i, 0, len(a) - 1)], 0).astype(np.float64)
        m = b[e].astype(np.float64).T if trans_b else b[e].astype(np.float64)
        out[for_rows] = alpha * (x @ m) + beta * c[for_rows]
        scale[for_rows] += abs(alpha) * (np.abs(x) @ np.abs(m))
    return out, scale


@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("size", GROUPED, ids=str)
def test_grouped_gemm(D, size, trans_b):
    groups, rows, k, n = size
    for turn, (kind, whole, alpha, beta) in enumerate((("any", True, 1.0, 0.0), ("one", False, 1.0, 0.0), ("short", True, 2.0, -1.0), ("any", False, -0.5, 0.75))):
        rng = np.random.default_rng(rows + k + turn)
        make = (lambda *s: rng.integers(-7, 8, s).astype(D.type)) if whole else (lambda *s: rng.standard_normal(s).astype(D.type))
        offsets = offsets_of(rng, groups, rows, kind)
        a_rows = rows if turn % 2 == 0 else max(1, rows // 2)
        index = np.arange(rows) if turn % 2 == 0 else rng.integers(0, a_rows, rows)
        if turn == 3:
            index[::5] = rng.choice([-1, a_rows, 1 << 30, -(1 << 31)], len(index[::5]))
        a, c = make(a_rows, k), make(rows, n)
        b = make(groups, n, k) if trans_b else make(groups, k, n)
        ta, tc = D.block(a, turn), D.block(c, turn % 3)
        blocks.grouped_gemm(tc, trans_b, alpha, ta, D.tensor(b), beta, D.tensor(offsets, "int"),
                            index=None if turn % 2 == 0 else D.tensor(index, "int"))
        want, scale = grouped64(a, index, b, trans_b, offsets, c, alpha, beta)
        got = read(tc)
        inside = np.zeros(rows, bool)
        inside[offsets[0]:offsets[-1]] = True
        assert np.array_equal(got[~inside], c[~inside]), "rows of no group were written"
        if whole:
            assert np.array_equal(got.astype(np.float64), want), (kind, capi.last_kernel())
        else:
            close(got, want, scale, (k + 4) * D.u, f"{kind} {capi.last_kernel()}")


@pytest.mark.parametrize("size", GROUPED, ids=str)
def test_grouped_gemm_weights(D, size):
    groups, rows, m, n = size
    for turn, (kind, whole, alpha, beta) in enumerate((("any", True, 1.0, 0.0), ("one", False, 1.0, 0.0), ("short", True, 2.0, -1.0), ("any", False, -0.5, 0.75))):
        rng = np.random.default_rng(rows + m + turn)
        make = (lambda *s: rng.integers(-7, 8, s).astype(D.type)) if whole else (lambda *s: rng.standard_normal(s).astype(D.type))
        offsets = offsets_of(rng, groups, rows, kind)
        a_rows, b_rows = (rows, rows) if turn == 0 else (max(1, rows // 2), rows + 3)
        ia, ib = (np.arange(rows),) * 2 if turn == 0 else (rng.integers(0, a_rows, rows), rng.integers(0, b_rows, rows))
        if turn == 3:
            ia[::4], ib[1::6] = -1, b_rows
        a, b, c = make(a_rows, m), make(b_rows, n), make(groups, m, n)
        ta, tb, tc = D.block(a, turn), D.block(b, turn + 1), D.tensor(c)
        indexes = {} if turn == 0 else {"a_index": D.tensor(ia, "int"), "b_index": D.tensor(ib, "int")}
        blocks.grouped_gemm_weights(tc, alpha, ta, tb, beta, D.tensor(offsets, "int"), **indexes)
        got = read(tc)
        rows_of = lambda x, i: np.where(((i >= 0) & (i < len(x)))[:, None], x[np.clip(i, 0, len(x) - 1)], 0).astype(np.float64)
        for e in range(groups):
            i = slice(offsets[e], offsets[e + 1])
            x, y = rows_of(a, ia[i]), rows_of(b, ib[i])
            want = alpha * (x.T @ y) + beta * c[e].astype(np.float64)
            if whole:
                assert np.array_equal(got[e].astype(np.float64), want), (kind, e, capi.last_kernel())
            else:
                close(got[e], want, abs(alpha) * (np.abs(x).T @ np.abs(y)) + np.abs(beta * c[e]), (len(x) + 4) * D.u, f"{kind} {capi.last_kernel()}")


@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("size", [(2, 300, 4100, 200), (1, 260, 2081, 65), (1, 900, 4129, 65), (8, 1100, 3000, 260)], ids=str)
def test_grouped_gemm_whose_sums_are_divided(stream, size, trans_b):
    """Few tiles and long sums: blocks take parts of k, and a second launch adds them up, in the groups' rows alone (not of 260
    rows by 65, which the kernel for a few rows takes)."""
    D = Owned("float")
    groups, rows, k, n = size
    for turn, (kind, whole, alpha, beta) in enumerate((("any", True, 1.0, 0.0), ("short", False, 1.5, 0.0), ("one", False, -0.5, 0.75))):
        rng = np.random.default_rng(rows + k + turn)
        make = (lambda *s: rng.integers(-7, 8, s).astype(np.float32)) if whole else (lambda *s: rng.standard_normal(s).astype(np.float32))
        offsets = offsets_of(rng, groups, rows, kind)
        index = rng.integers(0, rows, rows)
        index[::7] = rng.choice([-1, rows, 1 << 30], len(index[::7]))
        a, c = make(rows, k), make(rows, n)
        b = make(groups, n, k) if trans_b else make(groups, k, n)
        tc = D.block(c, turn)
        blocks.grouped_gemm(tc, trans_b, alpha, D.block(a, turn), D.tensor(b), beta, D.tensor(offsets, "int"), index=D.tensor(index, "int"))
        assert capi.last_kernel() == "grouped_thin" if rows == 260 else capi.last_kernel().endswith("+grouped_sum")
        want, scale = grouped64(a, index, b, trans_b, offsets, c, alpha, beta)
        got = read(tc)
        inside = np.zeros(rows, bool)
        inside[offsets[0]:offsets[-1]] = True
        assert np.array_equal(got[~inside], c[~inside]), "rows of no group were written"
        if whole:
            assert np.array_equal(got.astype(np.float64), want)
        else:
            close(got, want, scale, (k + 4) * 2.0 ** -24, kind)
    D.free()


@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("size", [(2, 9, 2500, 55), (29, 11, 2532, 55), (1, 40, 1031, 33), (3, 200, 4100, 70)], ids=str)
def test_grouped_gemm_in_double_whose_sums_are_divided(stream, size, trans_b):
    D = Owned("double")
    groups, rows, k, n = size
    for turn, (kind, whole, alpha, beta) in enumerate((("any", True, 1.0, 0.0), ("short", False, 1.5, 0.0), ("one", False, -0.5, 0.75))):
        rng = np.random.default_rng(rows + k + turn)
        make = (lambda *s: rng.integers(-7, 8, s).astype(np.float64)) if whole else (lambda *s: rng.standard_normal(s))
        offsets = offsets_of(rng, groups, rows, kind)
        index = rng.integers(0, rows, rows)
        index[::7] = rng.choice([-1, rows, 1 << 30], len(index[::7]))
        a, c = make(rows, k), make(rows, n)
        b = make(groups, n, k) if trans_b else make(groups, k, n)
        tc = D.block(c, turn)
        blocks.grouped_gemm(tc, trans_b, alpha, D.block(a, turn), D.tensor(b), beta, D.tensor(offsets, "int"), index=D.tensor(index, "int"))
        assert capi.last_kernel() == "grouped_double+grouped_sum"
        want, scale = grouped64(a, index, b, trans_b, offsets, c, alpha, beta)
        got = read(tc)
        inside = np.zeros(rows, bool)
        inside[offsets[0]:offsets[-1]] = True
        assert np.array_equal(got[~inside], c[~inside]), "rows of no group were written"
        if whole:
            assert np.array_equal(got, want)
        else:
            close(got, want, scale, (k + 4) * 2.0 ** -53, kind)
    D.free()


@pytest.mark.parametrize("size", [(2, 9000, 130, 70), (3, 7001, 33, 65), (1, 5000, 64, 64)], ids=str)
def test_grouped_gemm_weights_whose_sums_are_divided(D, size):
    groups, rows, m, n = size
    for turn, (kind, whole, alpha, beta) in enumerate((("any", True, 1.0, 0.0), ("short", False, 1.5, 0.0), ("one", False, -0.5, 0.75))):
        rng = np.random.default_rng(rows + m + turn)
        make = (lambda *s: rng.integers(-7, 8, s).astype(D.type)) if whole else (lambda *s: rng.standard_normal(s).astype(D.type))
        offsets = offsets_of(rng, groups, rows, kind)
        ia = rng.integers(0, rows, rows)
        ia[::9] = -1
        a, b, c = make(rows, m), make(rows, n), make(groups, m, n)
        tc = D.tensor(c)
        blocks.grouped_gemm_weights(tc, alpha, D.block(a, turn), D.block(b, 1), beta, D.tensor(offsets, "int"), a_index=D.tensor(ia, "int"))
        assert capi.last_kernel().endswith("+grouped_sum")
        got, x_all = read(tc), np.where((ia >= 0)[:, None], a[ia], 0).astype(np.float64)
        for e in range(groups):
            x, y = x_all[offsets[e]:offsets[e + 1]], b[offsets[e]:offsets[e + 1]].astype(np.float64)
            want = alpha * (x.T @ y) + beta * c[e].astype(np.float64)
            if whole:
                assert np.array_equal(got[e].astype(np.float64), want), (kind, e)
            else:
                close(got[e], want, abs(alpha) * (np.abs(x).T @ np.abs(y)) + np.abs(beta * c[e]), (len(x) + 4) * D.u, kind)


def test_grouped_gemm_weights_of_an_operand_beyond_four_gib(stream):
    """Rows that begin past 2^32 bytes are found: whole numbers, every sum exact."""
    D = Owned("float")
    rng = np.random.default_rng(35)
    ld, a_rows = 1 << 16, (1 << 14) + 40                      # 4.01 GiB of which 200 columns of a few rows are looked at
    rows, m, n = 300, 200, 70
    whole = ct.new_tensor([a_rows * ld], datatype="float")
    D.kept.append(whole)
    index = np.concatenate([rng.integers(0, 40, rows // 2), rng.integers(a_rows - 40, a_rows, rows - rows // 2)])
    small = rng.integers(-7, 8, (a_rows, m)).astype(np.float32)
    for r in np.unique(index):
        row = D.tensor(small[r])
        capi.call("ct_memcpy_async", whole.buffer.ptr + 4 * ld * int(r), row.buffer.ptr, 4 * m, capi.COPY_D2D, stream.handle)
    a = ct.Tensor(whole.device, {"shape": [a_rows, m], "strides": [ld, 1]}, whole.buffer)
    b = rng.integers(-7, 8, (rows, n)).astype(np.float32)
    offsets = np.array([0, 120, 120, rows])
    tc = D.tensor(np.zeros((3, m, n)))
    blocks.grouped_gemm_weights(tc, 1.0, a, D.tensor(b), 0.0, D.tensor(offsets, "int"), a_index=D.tensor(index, "int"))
    x = small[index].astype(np.float64)
    for e in range(3):
        i = slice(offsets[e], offsets[e + 1])
        assert np.array_equal(read(tc)[e].astype(np.float64), x[i].T @ b[i])
    # the same operand's rows in the products
    weights, c = rng.integers(-7, 8, (3, n, m)).astype(np.float32), D.tensor(np.zeros((rows, n)))
    blocks.grouped_gemm(c, True, 1.0, a, D.tensor(weights), 0.0, D.tensor(offsets, "int"), index=D.tensor(index, "int"))
    want, _ = grouped64(small, index, weights, True, offsets, np.zeros((rows, n), np.float32), 1.0, 0.0)
    assert np.array_equal(read(c).astype(np.float64), want)
    D.free()


def test_grouped_products_without_terms_or_rows(D, stream):
    """Sums of no terms, and operands without rows, whose indexes all lie outside: beta times what was there, in the groups' rows."""
    code = capi.DTYPE_CODES[D.datatype]
    rows, k, n = 9, 5, 6
    offsets, index = D.tensor([0, 4, 7], "int"), D.tensor(np.arange(rows), "int")
    b = D.tensor(np.ones((2, n, k)))
    for a_rows, terms in ((rows, 0), (0, k)):
        for beta in (0.0, 0.5):
            c = np.arange(rows * n, dtype=D.type).reshape(rows, n) + 1
            tc = D.tensor(c)
            capi.call("ct_grouped_gemm", stream.handle, tc.buffer.ptr, n, 1, 1.0, None, a_rows, terms, k, index.buffer.ptr, b.buffer.ptr, n, k,
                      n * k, offsets.buffer.ptr, 2, rows, beta, code)
            assert np.array_equal(read(tc), np.concatenate([beta * c[:7], c[7:]]))
    y = D.tensor(np.ones((rows, n)))
    for beta in (0.0, 0.5):
        w = np.arange(2 * k * n, dtype=D.type).reshape(2, k, n) + 1
        tw = D.tensor(w)
        capi.call("ct_grouped_gemm_weights", stream.handle, tw.buffer.ptr, n, k * n, 1.0, None, 0, k, k, index.buffer.ptr, y.buffer.ptr, rows, n, n,
                  None, offsets.buffer.ptr, 2, rows, beta, code)
        assert np.array_equal(read(tw), beta * w)


def test_grouped_products_of_rows_far_apart(stream):
    """Further than the tiles' 32-bit offsets reach: a matrix's rows 2^22 floats and more apart, and operands of the weights' products
    2^30 and more.  Whole numbers: every sum exact."""
    D = Owned("float")
    rng = np.random.default_rng(53)
    rows, k, n, ld = 200, 64, 5, (1 << 22) + 3
    a, b = rng.integers(-7, 8, (rows, k)).astype(np.float32), rng.integers(-7, 8, (n, k)).astype(np.float32)
    far = ct.new_tensor([n * ld], datatype="float")
    D.kept.append(far)
    for r in range(n):
        row = D.tensor(b[r])
        capi.call("ct_memcpy_async", far.buffer.ptr + 4 * ld * r, row.buffer.ptr, 4 * k, capi.COPY_D2D, stream.handle)
    offsets, c = D.tensor([0, rows], "int"), D.tensor(np.zeros((rows, n)))
    capi.call("ct_grouped_gemm", stream.handle, c.buffer.ptr, n, 1, 1.0, D.tensor(a).buffer.ptr, rows, k, k, None, far.buffer.ptr, n, ld, n * ld,
              offsets.buffer.ptr, 1, rows, 0.0, capi.F32)
    assert np.array_equal(read(c), a @ b.T)
    ld = (1 << 30) + 5
    x, y = rng.integers(-7, 8, (2, 70)).astype(np.float32), rng.integers(-7, 8, (2, 33)).astype(np.float32)
    far = ct.new_tensor([ld + 70], datatype="float")
    D.kept.append(far)
    for r in range(2):
        row = D.tensor(x[r])
        capi.call("ct_memcpy_async", far.buffer.ptr + 4 * ld * r, row.buffer.ptr, 4 * 70, capi.COPY_D2D, stream.handle)
    offsets, w = D.tensor([0, 2], "int"), D.tensor(np.zeros((1, 70, 33)))
    capi.call("ct_grouped_gemm_weights", stream.handle, w.buffer.ptr, 33, 70 * 33, 1.0, far.buffer.ptr, 2, 70, ld, None, D.tensor(y).buffer.ptr, 2, 33, 33,
              None, offsets.buffer.ptr, 1, 2, 0.0, capi.F32)
    assert np.array_equal(read(w)[0], x.T @ y)
    D.free()


def test_grouped_offsets_that_make_no_sense_stay_inside(D):
    """Offsets that decrease or lie outside the rows are clamped: whatever is computed, nothing beside the result changes."""
    rng = np.random.default_rng(31)
    a, b = rng.standard_normal((50, 40)), rng.standard_normal((3, 30, 40))
    for offsets in ([0, 60, 20, 1000], [-5, -1, 90, 3], [50, 50, 50, 50], [2 ** 31 - 1, -2 ** 31, 0, 7]):
        tc, tw = D.block(np.zeros((50, 30)), 2), D.tensor(np.zeros((3, 40, 30)))
        t = D.tensor(np.array(offsets), "int")
        blocks.grouped_gemm(tc, True, 1.0, D.tensor(a), D.tensor(b), 0.0, t)
        blocks.grouped_gemm_weights(tw, 1.0, D.tensor(a), D.tensor(rng.standard_normal((50, 30))), 0.0, t)
        assert np.all(np.isfinite(read(tc))) and np.all(np.isfinite(read(tw)))


def test_grouped_products_of_what_is_not_finite(stream):
    """Infinities, NaN and floats near the ends of their range: the same classes as the sum of the products has, and the
    other rows and groups untouched by them."""
    D = Owned("float")
    rng = np.random.default_rng(32)
    for rows, k, n in ((40, 50, 60), (300, 200, 260), (9, 400, 100)):
        a, b = rng.standard_normal((rows, k)).astype(np.float32), rng.standard_normal((2, n, k)).astype(np.float32)
        a[1, 3], a[2, 0], a[3, k - 1] = np.inf, np.nan, 3e38
        a[4] *= np.float32(1e-38)
        b[1, 5, 2] = -np.inf
        offsets = np.array([0, rows // 2, rows])
        tc = D.tensor(np.zeros((rows, n)))
        blocks.grouped_gemm(tc, True, 1.0, D.tensor(a), D.tensor(b), 0.0, D.tensor(offsets, "int"))
        with np.errstate(all="ignore"):
            want, scale = grouped64(a, np.arange(rows), b, True, offsets, np.zeros((rows, n), np.float32), 1.0, 0.0)
        got = read(tc).astype(np.float64)
        sure = ~(scale > 1e38) | np.isinf(scale)   # a sum that comes near the largest float may pass it on the way
        for cls in (np.isnan, np.isposinf, np.isneginf):
            assert np.array_equal(cls(got)[sure], cls(want)[sure])
        fine = sure & np.isfinite(want)
        assert np.all(np.abs(got - want)[fine] <= ((k + 4) * 2.0 ** -24 * scale + k * 2.0 ** -149)[fine])
    D.free()


# ------------------------------------------------------------------------------------------------- combining

COMBINE = [(1, 1, 1), (3, 2, 5), (17, 8, 130), (64, 3, 64), (5, 32, 257), (40, 4, 1000), (9, 9, 1031), (300, 2, 2048), (2, 5, 5000)]


@pytest.mark.parametrize("size", COMBINE, ids=str)
def test_combine_experts(D, size):
    n, k, width = size
    rng = np.random.default_rng(n + width)
    for turn in range(2):
        count = n * k + turn
        slots = rng.permutation(count)[:n * k].reshape(n, k)
        if turn:
            lost = rng.random((n, k)) < 0.3
            lost[n // 2] = True                       # a token without any row
            slots = np.where(lost, rng.choice([-1, count, 1 << 30, -(1 << 31)], (n, k)), slots)
        have = (slots >= 0) & (slots < count)
        rows, weights, dy = (rng.standard_normal(s).astype(D.type) for s in ((count, width), (n, k), (n, width)))
        rows[np.setdiff1d(np.arange(count), slots[have])] = np.nan      # no token's: never read
        tr, tw, ts = D.block(rows, turn), D.tensor(weights), D.tensor(slots, "int")
        taken = np.where(have[:, :, None], rows[np.where(have, slots, 0)].astype(np.float64), 0)
        for w, given in ((weights.astype(np.float64), tw), (np.ones((n, k)), None)):
            out = D.block(np.zeros((n, width)), 1)
            blocks.combine_experts(out, tr, given, ts)
            terms = w[:, :, None] * taken
            close(read(out), terms.sum(1), np.abs(terms).sum(1), (k + 4) * D.u, "output")
            to, dw = D.block(np.full((count, width), 5.0), 2), D.tensor(np.full((n, k), 9.0))
            blocks.combine_experts_gradient(to, dw, D.block(dy, 3), tr, given, ts)
            want = np.full((count, width), 5.0)
            for t, j in zip(*np.nonzero(have)):
                want[slots[t, j]] = (D.type(w[t, j]) * dy[t])
            assert np.array_equal(read(to), want.astype(D.type)), "rows gradient"
            dots = taken * dy[:, None, :].astype(np.float64)
            close(read(dw), dots.sum(2), np.abs(dots).sum(2), (width + 4) * D.u, "weights gradient")
    # one of the two
    dw2, to2 = D.tensor(np.zeros((n, k))), D.tensor(np.full((count, width), 5.0))
    blocks.combine_experts_gradient(None, dw2, D.tensor(dy), tr, None, ts)
    blocks.combine_experts_gradient(to2, None, D.tensor(dy), None, None, ts)
    assert np.array_equal(read(dw2), read(dw)) and np.array_equal(read(to2), read(to))


def test_combine_of_rows_without_elements(D):
    """Nothing to add up: the weights' gradient is zero, and nothing else is written."""
    dw, ts = D.tensor(np.full((5, 2), 9.0)), D.tensor(np.arange(10).reshape(5, 2), "int")
    empty = lambda n: D.tensor(np.zeros((n, 0)))
    blocks.combine_experts(empty(5), empty(10), None, ts)
    blocks.combine_experts_gradient(empty(10), dw, empty(5), empty(10), None, ts)
    assert np.all(read(dw) == 0)


# ------------------------------------------------------------------------------------------------- clipping

@pytest.mark.parametrize("sizes", [[1], [3, 0, 5], [100352, 128, 1280, 10], [16384, 16385, 1, 32767, 40001], list(range(1, 260)),
                                   [70000] * 9, [0, 0]], ids=lambda s: f"{len(s)} of {max(s)}")
def test_clip_gradients(D, sizes, stream):
    rng = np.random.default_rng(len(sizes))
    host = [(rng.standard_normal(n) * 10.0 ** rng.uniform(-3, 1)).astype(D.type) for n in sizes]
    norm64 = np.sqrt(sum((h.astype(np.float64) ** 2).sum() for h in host))
    backend = optimize.Backend(stream, D.datatype)
    n = sum(sizes)
    bar = 4 * D.u + max(n, 1) * 2.0 ** -53
    for limit in (norm64 * 0.25 if norm64 else 1.0, norm64 * 4 + 1, float("inf")):
        # the gradients side by side behind one element, so that none keeps to the 16-byte grid
        flat = D.tensor(np.concatenate([[7.25]] + host + [[7.25]]))
        into = D.tensor(np.full(n + 3, 7.25))
        result = D.tensor(np.zeros(2))
        ends = np.cumsum([1] + sizes)
        gradients = [flat.buffer.sub_buffer(int(a), s) for a, s in zip(ends, sizes)]
        outputs = [into.buffer.sub_buffer(int(a) + 1, s) for a, s in zip(ends, sizes)]
        optimize.clip_gradients(backend, gradients, limit, result, outputs)
        norm, factor = read(result)
        want = min(1.0, limit / norm64) if norm64 else 1.0
        assert abs(float(norm) - norm64) <= bar * norm64 and abs(float(factor) - want) <= bar * want
        clipped = np.concatenate([[7.25] * 2] + [h * factor for h in host] + [[7.25]]).astype(D.type)
        assert np.array_equal(read(into), clipped)
        # the norm alone, then in place: the same bits
        before = read(flat)
        result2 = D.tensor(np.zeros(2))
        optimize.clip_gradients(backend, gradients, limit, result2, in_place=False)
        assert np.array_equal(read(result2), read(result)) and np.array_equal(read(flat), before)
        optimize.clip_gradients(backend, gradients, limit, result2)
        assert np.array_equal(read(result2), read(result))
        assert np.array_equal(read(flat), np.concatenate([[7.25]] + [h * factor for h in host] + [[7.25]]).astype(D.type))


def test_clip_gradients_beyond_the_square_root_of_the_range(stream):
    """Squares of floats that a float does not hold."""
    D = Owned("float")
    backend = optimize.Backend(stream, "float")
    for x in (1e30, 1e-30):
        t, result = D.tensor(np.full(1000, x)), D.tensor(np.zeros(2))
        optimize.clip_gradients(backend, [t], 1e-31, result)
        norm, factor = read(result)
        want = np.sqrt(1000 * float(np.float32(x)) ** 2)
        assert abs(norm - want) <= 1e-6 * want and abs(factor - 1e-31 / want) <= 1e-6 * (1e-31 / want) + 2.0 ** -149
    D.free()


def test_clip_gradients_that_are_not_finite(D, stream):
    backend = optimize.Backend(stream, D.datatype)
    for bad in (np.nan, np.inf):
        t, result = D.tensor(np.array([1.0, bad, 2.0])), D.tensor(np.zeros(2))
        optimize.clip_gradients(backend, [t], 1.0, result)
        norm, factor = read(result)
        got = read(t)
        if np.isnan(bad):
            assert np.isnan(norm) and np.isnan(factor) and np.all(np.isnan(got))
        else:
            assert np.isinf(norm) and factor == 0 and got[0] == 0 and got[2] == 0 and np.isnan(got[1])


# ------------------------------------------------------------------------------------------------- the checks in Python

def test_operands_that_only_the_checks_in_python_take(stream, monkeypatch):
    """Every call comes out the same whether its operands are found in native code or by the checks behind it."""
    D = Owned("float")
    n, width, experts, chosen = 37, 24, 6, 2

    def run():
        random = np.random.default_rng(48)
        make = lambda *s: D.tensor(random.standard_normal(s))
        empty, whole = (lambda *s: D.tensor(np.zeros(s))), (lambda *s: D.tensor(np.zeros(s), "int"))
        x, residual, h, out, statistics = make(n, width), make(n, width), empty(n, width), empty(n, width), empty(4, n)
        p = {"pre-scale": make(width), "post-scale": make(width), "gate": make(1, width)}
        g = {k: empty(*t.shape()) for k, t in p.items()}
        d = blocks.norm_descriptor(post="rms", pre="rms")
        blocks.norm_residual(out, h, statistics, x, residual, p, d)
        dx, dr = empty(n, width), empty(n, width)
        blocks.norm_residual_gradient(dx, dr, g, make(n, width), make(n, width), x, out, statistics, p, d)
        at, w, offsets, tokens, slots = whole(n, chosen), empty(n, chosen), whole(experts + 1), whole(n * chosen), whole(n, chosen)
        logits, dl = make(n, experts), empty(n, experts)
        blocks.route_experts(at, w, offsets, tokens, slots, logits)
        blocks.route_experts_gradient(dl, make(n, chosen), w, at, logits)
        rows, dw = empty(n * chosen, width), empty(experts, width, width)
        blocks.grouped_gemm(rows, True, 1.0, h, make(experts, width, width), 0.0, offsets, index=tokens)
        blocks.grouped_gemm_weights(dw, 1.0, rows, h, 0.0, offsets, b_index=tokens)
        y, drows, dweights = empty(n, width), empty(n * chosen, width), empty(n, chosen)
        blocks.combine_experts(y, rows, w, slots)
        blocks.combine_experts_gradient(drows, dweights, make(n, width), rows, w, slots)
        norm = empty(2)
        optimize.clip_gradients(optimize.Backend(stream), [dw, drows], 1.0, norm)
        return [read(t) for t in (out, h, dx, dr, *g.values(), at, w, offsets, tokens, slots, dl, rows, dw, y, drows, dweights, norm)]

    found = run()
    monkeypatch.setattr(blocks, "_operands", lambda kinds, tensors: None)
    for a, b in zip(found, run()):
        assert np.array_equal(a, b)
    D.free()


# ------------------------------------------------------------------------------------------------- graphs

def test_calls_recorded_into_a_graph(as_released):
    """A step of every operator, recorded with the scratch that the stream holds and replayed with new inputs, eager calls of
    the same step in between: each replay's results are the eager ones, bit for bit."""
    import ctypes as C
    rt = C.CDLL("libamdhip64.so")
    stream = drv.HipDriver().default_device().create_stream()
    D = Owned("float")
    rng = np.random.default_rng(43)
    width, experts, chosen, inner = 200, 6, 2, 2100
    with ct.tensor_context(stream, "float"):
        make = lambda *s: D.tensor(rng.standard_normal(s))
        sides = []
        p = {"pre-scale": make(width), "pre-bias": make(width), "post-scale": make(width), "post-bias": make(width), "gate": make(1, width)}
        inputs = {n: {"x": make(n, width), "r": make(n, width), "do": make(n, width), "dh": make(n, width), "logits": make(n, experts),
                      "dw": make(n, chosen), "y": make(n * chosen, inner), "dy": make(n, width)} for n in (100, 1300)}
        first, second = make(experts, inner, width), make(experts, width, inner)
        for _ in range(2):
            side = {"norm": D.tensor(np.zeros(2))}
            for n in inputs:
                empty, whole = (lambda *s: D.tensor(np.zeros(s))), (lambda *s: D.tensor(np.zeros(s), "int"))
                side[n] = dict(out=empty(n, width), h=empty(n, width), statistics=empty(4, n), dx=empty(n, width), dr=empty(n, width),
                               g={k: empty(*t.shape()) for k, t in p.items()}, at=whole(n, chosen), w=empty(n, chosen), offsets=whole(experts + 1),
                               tokens=whole(n * chosen), slots=whole(n, chosen), dl=empty(n, experts), rows=empty(n * chosen, inner),
                               back=empty(n * chosen, width), d_first=empty(experts, inner, width), y=empty(n, width),
                               d_back=empty(n * chosen, width), d_weights=empty(n, chosen))
            sides.append(side)

        d = blocks.norm_descriptor(post="layer", pre="layer", residual_scale=0.5)

        def step(side):
            for n, i in inputs.items():
                o = side[n]
                blocks.norm_residual(o["out"], o["h"], o["statistics"], i["x"], i["r"], p, d)
                blocks.norm_residual_gradient(o["dx"], o["dr"], o["g"], i["do"], i["dh"], i["x"], o["out"], o["statistics"], p, d)
                blocks.route_experts(o["at"], o["w"], o["offsets"], o["tokens"], o["slots"], i["logits"])
                blocks.route_experts_gradient(o["dl"], i["dw"], o["w"], o["at"], i["logits"])
                blocks.grouped_gemm(o["rows"], True, 1.0, o["h"], first, 0.0, o["offsets"], index=o["tokens"])
                blocks.grouped_gemm(o["back"], True, 1.0, i["y"], second, 0.0, o["offsets"])
                blocks.grouped_gemm_weights(o["d_first"], 1.0, o["rows"], o["h"], 0.0, o["offsets"], b_index=o["tokens"])
                blocks.combine_experts(o["y"], o["back"], o["w"], o["slots"])
                blocks.combine_experts_gradient(o["d_back"], o["d_weights"], i["dy"], o["back"], o["w"], o["slots"])
            optimize.clip_gradients(optimize.Backend(stream), [t for n in inputs for t in side[n]["g"].values()] + [side[n]["d_first"] for n in inputs],
                                    1.0, side["norm"])

        def results(side):
            out = [read(side["norm"])]
            for n in inputs:
                for t in side[n].values():
                    out += [read(v) for v in (t.values() if isinstance(t, dict) else [t])]
            return out

        step(sides[1])      # kernels are loaded and scratch is in place
        capi.call("ct_stream_sync", stream.handle)
        graph, graph_exec = C.c_void_p(), C.c_void_p()
        rt.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
        rt.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
        rt.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
        rt.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
        rt.hipGraphExecDestroy.argtypes = rt.hipGraphDestroy.argtypes = [C.c_void_p]
        assert rt.hipStreamBeginCapture(stream.handle, 1) == 0
        try:
            step(sides[1])
        finally:
            ended = rt.hipStreamEndCapture(stream.handle, C.byref(graph))
        assert ended == 0 and graph.value
        assert rt.hipGraphInstantiate(C.byref(graph_exec), graph, None, None, 0) == 0
        for replay in range(4):
            for n, i in inputs.items():
                for t in i.values():
                    new = D.tensor(rng.standard_normal(t.shape()))
                    capi.call("ct_memcpy_async", t.buffer.ptr, new.buffer.ptr, t.ecount() * 4, capi.COPY_D2D, stream.handle)
            step(sides[0])
            want = results(sides[0])
            assert rt.hipGraphLaunch(graph_exec, stream.handle) == 0
            for a, b in zip(results(sides[1]), want):
                assert np.all(np.isfinite(b)) and np.array_equal(a, b), replay
        capi.call("ct_stream_sync", stream.handle)
        assert rt.hipGraphExecDestroy(graph_exec) == 0 and rt.hipGraphDestroy(graph) == 0
        D.free()
    stream.release()


def test_divided_sums_recorded_without_scratch_do_without(as_released):
    """A capture that finds no scratch for the parts: one launch, and the same whole numbers."""
    import ctypes as C
    rt = C.CDLL("libamdhip64.so")
    rt.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    rt.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    rt.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    rt.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    rt.hipGraphExecDestroy.argtypes = rt.hipGraphDestroy.argtypes = [C.c_void_p]
    rng = np.random.default_rng(45)
    for datatype in ("float", "double"):
        D = Owned(datatype)
        device = drv.HipDriver().default_device()
        stream, loader = device.create_stream(), device.create_stream()
        make = lambda *s: rng.integers(-7, 8, s).astype(NUMPY[datatype])
        a, b, x = make(300, 4100), make(2, 200, 4100), make(300, 64)
        offsets = np.array([0, 140, 300])
        with ct.tensor_context(loader, datatype):
            ta, tb, tx, to = D.tensor(a), D.tensor(b), D.tensor(x), D.tensor(offsets, "int")
            tc, tw = D.tensor(np.zeros((300, 200))), D.tensor(np.zeros((2, 64, 64)))
            long, wide = D.tensor(make(9000, 64)), D.tensor(np.array([0, 5000, 9000]), "int")
            blocks.grouped_gemm(tc, True, 1.0, ta, tb, 0.0, to)        # the kernels are loaded
            blocks.grouped_gemm_weights(tw, 1.0, long, long, 0.0, wide)
            assert capi.last_kernel().endswith("+grouped_sum")
            capi.call("ct_stream_sync", loader.handle)
        kernels = []
        with ct.tensor_context(stream, datatype):
            graph, graph_exec = C.c_void_p(), C.c_void_p()
            assert rt.hipStreamBeginCapture(stream.handle, 1) == 0
            try:
                blocks.grouped_gemm(tc, True, 1.0, ta, tb, 0.0, to)
                kernels.append(capi.last_kernel())
                blocks.grouped_gemm_weights(tw, 1.0, long, long, 0.0, wide)
                kernels.append(capi.last_kernel())
            finally:
                ended = rt.hipStreamEndCapture(stream.handle, C.byref(graph))
            assert ended == 0 and graph.value and not any(k.endswith("+grouped_sum") for k in kernels), kernels
            assert rt.hipGraphInstantiate(C.byref(graph_exec), graph, None, None, 0) == 0
            host = read(long).astype(np.float64)
            for _ in range(2):
                assert rt.hipGraphLaunch(graph_exec, stream.handle) == 0
                got, weights = read(tc).astype(np.float64), read(tw).astype(np.float64)
                for e in range(2):
                    i, j = slice(offsets[e], offsets[e + 1]), slice(*((0, 5000), (5000, 9000))[e])
                    assert np.array_equal(got[i], a[i].astype(np.float64) @ b[e].T.astype(np.float64))
                    assert np.array_equal(weights[e], host[j].T @ host[j])
            capi.call("ct_stream_sync", stream.handle)
            assert rt.hipGraphExecDestroy(graph_exec) == 0 and rt.hipGraphDestroy(graph) == 0
            D.free()
        stream.release()
        loader.release()


# ------------------------------------------------------------------------------------------------- streams

def test_calls_on_two_streams_do_not_meet(as_released):
    """Each stream has its own scratch memory: the same calls on two streams at once give what each gives alone."""
    device = drv.HipDriver().default_device()
    rng = np.random.default_rng(41)
    results = []
    D = Owned("float")
    streams = [device.create_stream() for _ in range(2)]
    data = [rng.standard_normal((3000, 64)).astype(np.float32) for _ in range(2)]
    made = []
    for s, x in zip(streams, data):
        with ct.tensor_context(s, "float"):
            made.append([D.tensor(x), D.tensor(np.zeros((3000, 4)), "int"), D.tensor(np.zeros((3000, 4))), D.tensor(np.zeros(65), "int"),
                         D.tensor(np.zeros(12000), "int"), D.tensor(np.zeros((3000, 4)), "int"), D.tensor(np.zeros(2))])
    for _ in range(20):
        for s, (t, experts, weights, offsets, tokens, slots, norm) in zip(streams, made):
            with ct.tensor_context(s, "float"):
                blocks.route_experts(experts, weights, offsets, tokens, slots, t)
                optimize.clip_gradients(optimize.Backend(s), [t], 1.0, norm, in_place=False)
    for s, x, (t, experts, weights, offsets, tokens, slots, norm) in zip(streams, data, made):
        with ct.tensor_context(s, "float"):
            want = route64(x, 4, True)
            for got, w in ((experts, want[0]), (offsets, want[2]), (tokens, want[3]), (slots, want[4])):
                assert np.array_equal(read(got), w)
            assert abs(read(norm)[0] - np.linalg.norm(x.astype(np.float64))) <= 1e-6 * np.linalg.norm(x)
    D.free()
    for s in streams:
        s.release()
