"""What the operators of residual blocks with experts refuse: arguments are checked on the host, before any device call, in
the library and in the tensor API.  Nothing here needs a GPU."""
import ctypes as C

import pytest

from cortex_amd import blocks
from cortex_amd import capi
from cortex_amd import dimensions as dims
from cortex_amd import optimize
from cortex_amd import tensor as ct

F = capi.F32
A = [0x100000 + 0x100000 * i for i in range(24)]     # addresses that nothing follows


def refuses(message, name, *args):
    with pytest.raises(capi.CortexHipError) as e:
        capi.call(name, *args)
    assert e.value.status == 1 and message in e.value.message, e.value.message


def d(*shape, strides=None):
    return C.byref(capi.make_dims(shape, strides or dims.dimensions(list(shape))["strides"]))


def norm(rows=4, width=8, **change):
    args = dict(stream=None, output=A[0], output_dims=d(rows, width), normalized=A[1], normalized_dims=d(rows, width), statistics=A[2],
                input=A[3], input_dims=d(rows, width), residual=A[4], residual_dims=d(rows, width), gate=A[5], gate_dims=d(1, width),
                post_scale=A[6], post_bias=None, pre_scale=A[7], pre_bias=None, post_kind=1, pre_kind=1, residual_scale=1.0, epsilon=1e-5,
                dtype=F)
    args.update(change)
    return list(args.values())


@pytest.mark.parametrize("message,change", [
    ("float or double", {"dtype": capi.I32}), ("unknown kind", {"post_kind": 3}), ("unknown kind", {"pre_kind": -1}),
    ("epsilon", {"epsilon": -1.0}), ("epsilon", {"epsilon": float("nan")}), ("null buffer", {"input": None}),
    ("null buffer", {"normalized": None}), ("is needed", {"input_dims": d(4, 9)}), ("is needed", {"residual_dims": d(3, 8)}),
    ("innermost stride", {"input_dims": d(4, 8, strides=[1, 4])}), ("column stride", {"input_dims": d(4, 8, strides=[7, 1])}),
    ("is needed", {"gate_dims": d(2, 8)}), ("one or two", {"gate_dims": d(1, 1, 8)}), ("overlaps an operand", {"output": A[3] + 32}),
    ("overlaps an operand", {"output": A[5]}), ("results overlap", {"normalized": A[0]}), ("overlaps an operand", {"normalized": A[2]}),
    ("overlaps an operand", {"output": A[3], "output_dims": d(4, 8, strides=[16, 1])})])
def test_norm_residual(message, change):
    refuses(message, "ct_norm_residual", *norm(**change))


def norm_gradient(rows=4, width=8, **change):
    m = d(rows, width)
    args = dict(stream=None, input_gradient=A[0], input_gradient_dims=m, residual_gradient=A[1], residual_gradient_dims=m, gate_gradient=A[2],
                post_scale_gradient=A[3], post_bias_gradient=None, pre_scale_gradient=A[4], pre_bias_gradient=None, output_gradient=A[5],
                output_gradient_dims=m, normalized_gradient=A[6], normalized_gradient_dims=m, input=A[7], input_dims=m, output=A[8],
                output_dims=m, statistics=A[9], gate=A[10], gate_dims=d(1, width), post_scale=A[11], post_bias=None, pre_scale=A[12],
                post_kind=1, pre_kind=1, residual_scale=1.0, dtype=F)
    args.update(change)
    return list(args.values())


@pytest.mark.parametrize("message,change", [
    ("float or double", {"dtype": capi.I8}), ("unknown kind", {"post_kind": 7}), ("null buffer", {"input": None}),
    ("null buffer", {"statistics": None}), ("null buffer", {"output": None}), ("no gate", {"gate": None}),
    ("no post norm", {"post_kind": 0}), ("no pre norm", {"pre_kind": 0}), ("is needed", {"output_gradient_dims": d(4, 7)}),
    ("results overlap", {"residual_gradient": A[0]}), ("overlaps an operand", {"input_gradient": A[7]}),
    ("overlaps an operand", {"residual_gradient": A[5] + 4}), ("gate's gradient overlaps", {"gate_gradient": A[10]})])
def test_norm_residual_gradient(message, change):
    refuses(message, "ct_norm_residual_gradient", *norm_gradient(**change))


def route(**change):
    args = dict(stream=None, experts=A[0], weights=A[1], offsets=A[2], tokens=A[3], slots=A[4], logits=A[5], logits_colstride=16, n=10,
                n_experts=16, n_chosen=4, renormalize=1, dtype=F)
    args.update(change)
    return list(args.values())


@pytest.mark.parametrize("message,change", [
    ("float or double", {"dtype": capi.I64}), ("negative count", {"n": -1}), ("experts, 1 to", {"n_experts": 0}),
    ("experts, 1 to", {"n_experts": 1025, "logits_colstride": 1025}), ("chosen of", {"n_chosen": 0}), ("chosen of", {"n_chosen": 17}),
    ("chosen of", {"n_experts": 64, "n_chosen": 33, "logits_colstride": 64}), ("tokens", {"n": 1 << 30}), ("null buffer", {"logits": None}),
    ("null buffer", {"offsets": None}), ("column stride", {"logits_colstride": 15})])
def test_route_experts(message, change):
    refuses(message, "ct_route_experts", *route(**change))


def route_gradient(**change):
    args = dict(stream=None, logits_gradient=A[0], logits_gradient_colstride=16, weights_gradient=A[1], weights=A[2], experts=A[3],
                logits=A[4], logits_colstride=16, n=10, n_experts=16, n_chosen=4, renormalize=0, dtype=F)
    args.update(change)
    return list(args.values())


@pytest.mark.parametrize("message,change", [
    ("float or double", {"dtype": capi.U8}), ("negative count", {"n": -1}), ("chosen of", {"n_chosen": 17}), ("null buffer", {"logits": None}),
    ("null buffer", {"weights": None}), ("column stride", {"logits_gradient_colstride": 3}), ("column stride", {"logits_colstride": 3})])
def test_route_experts_gradient(message, change):
    refuses(message, "ct_route_experts_gradient", *route_gradient(**change))


def grouped(**change):
    args = dict(stream=None, c=A[0], c_colstride=32, trans_b=1, alpha=1.0, a=A[1], a_row_count=20, a_col_count=16, a_colstride=16, index=None,
                b=A[2], b_col_count=32, b_colstride=16, b_stride=512, offsets=A[3], n_groups=3, row_count=20, beta=0.0, dtype=F)
    args.update(change)
    return list(args.values())


@pytest.mark.parametrize("message,change", [
    ("float or double", {"dtype": capi.I16}), ("bad extent", {"row_count": -1}), ("bad extent", {"a_col_count": 1 << 31}),
    ("groups, at most", {"n_groups": 1 << 20}), ("null buffer", {"c": None}), ("null buffer", {"offsets": None}), ("null buffer", {"b": None}),
    ("rows of", {"a_row_count": 19}), ("column stride", {"c_colstride": 31}), ("column stride", {"a_colstride": 15}),
    ("column stride", {"b_colstride": 15}), ("column stride", {"trans_b": 0}), ("negative stride", {"b_stride": -1}),
    ("overlaps", {"c": A[1] + 64}), ("overlaps", {"c": A[2] + 4})])
def test_grouped_gemm(message, change):
    refuses(message, "ct_grouped_gemm", *grouped(**change))


def weights(**change):
    args = dict(stream=None, c=A[0], c_colstride=32, c_stride=512, alpha=1.0, a=A[1], a_row_count=20, a_col_count=16, a_colstride=16,
                a_index=None, b=A[2], b_row_count=20, b_col_count=32, b_colstride=32, b_index=None, offsets=A[3], n_groups=3, row_count=20,
                beta=0.0, dtype=F)
    args.update(change)
    return list(args.values())


@pytest.mark.parametrize("message,change", [
    ("float or double", {"dtype": capi.I16}), ("bad extent", {"b_row_count": -1}), ("groups, at most", {"n_groups": 1 << 20}),
    ("null buffer", {"a": None}), ("null buffer", {"c": None}), ("fewer rows", {"a_row_count": 19}), ("fewer rows", {"b_row_count": 19}),
    ("column stride", {"b_colstride": 31}), ("overlap one another", {"c_stride": 511}), ("c overlaps", {"c": A[2]})])
def test_grouped_gemm_weights(message, change):
    refuses(message, "ct_grouped_gemm_weights", *weights(**change))


def combine(**change):
    args = dict(stream=None, output=A[0], output_colstride=8, rows=A[1], row_count=20, rows_colstride=8, weights=A[2], slots=A[3], n=10,
                n_chosen=2, width=8, dtype=F)
    args.update(change)
    return list(args.values())


@pytest.mark.parametrize("message,change", [
    ("float or double", {"dtype": capi.I16}), ("bad extent", {"n": -1}), ("chosen, 1 to", {"n_chosen": 0}), ("chosen, 1 to", {"n_chosen": 33}),
    ("tokens", {"n": 1 << 30, "n_chosen": 4}), ("null buffer", {"slots": None}), ("null buffer", {"rows": None}),
    ("column stride", {"rows_colstride": 7}), ("overlap", {"output": A[1] + 32})])
def test_combine_experts(message, change):
    refuses(message, "ct_combine_experts", *combine(**change))


def combine_gradient(**change):
    args = dict(stream=None, rows_gradient=A[0], rows_gradient_colstride=8, weights_gradient=A[1], output_gradient=A[2],
                output_gradient_colstride=8, rows=A[3], row_count=20, rows_colstride=8, weights=A[4], slots=A[5], n=10, n_chosen=2, width=8,
                dtype=F)
    args.update(change)
    return list(args.values())


@pytest.mark.parametrize("message,change", [
    ("float or double", {"dtype": capi.I16}), ("bad extent", {"width": -1}), ("chosen, 1 to", {"n_chosen": 33}), ("null buffer", {"rows": None}),
    ("null buffer", {"output_gradient": None}), ("column stride", {"output_gradient_colstride": 7}),
    ("overlaps an operand", {"rows_gradient": A[2]}), ("overlaps an operand", {"rows_gradient": A[3] + 4})])
def test_combine_experts_gradient(message, change):
    refuses(message, "ct_combine_experts_gradient", *combine_gradient(**change))


def test_clip_gradients():
    def clip(gradients, outputs, counts, max_norm=1.0, result=A[9], dtype=F, count=None):
        g = (C.c_void_p * 4)(*gradients)
        o = (C.c_void_p * 4)(*outputs) if outputs is not None else None
        n = (C.c_int64 * 4)(*counts)
        return (None, g, o, n, len(gradients) if count is None else count, max_norm, result, dtype)
    refuses("float or double", "ct_clip_gradients", *clip([A[0]], None, [4], dtype=capi.I32))
    refuses("must be positive", "ct_clip_gradients", *clip([A[0]], None, [4], max_norm=0.0))
    refuses("must be positive", "ct_clip_gradients", *clip([A[0]], None, [4], max_norm=float("nan")))
    refuses("negative count", "ct_clip_gradients", *clip([A[0]], None, [4], count=-1))
    refuses("null argument", "ct_clip_gradients", *clip([A[0]], None, [4], result=None))
    refuses("tensor 1 has -4", "ct_clip_gradients", *clip([A[0], A[1]], None, [4, -4]))
    refuses("null buffer", "ct_clip_gradients", *clip([A[0], None], None, [4, 4]))
    refuses("null buffer", "ct_clip_gradients", *clip([A[0]], [None], [4]))
    refuses("overlaps its gradient", "ct_clip_gradients", *clip([A[0]], [A[0] + 4], [4]))


# ---------------------------------------------------------------- the tensor API

class Stub:
    """Stands in for a buffer, a device and a stream: whatever reaches the stream was not refused."""

    def __init__(self, ecount=0, datatype="float", ptr=0):
        self._ecount, self.datatype, self.ptr = ecount, datatype, ptr

    def ecount(self):
        return self._ecount

    def get_datatype(self):
        return self.datatype

    def partially_alias(self, other):
        return False

    def __getattr__(self, name):
        def call(*args):
            raise AssertionError(f"{name} was called")
        return call


DEVICE = object()


def t(*shape, datatype="float", strides=None, device=DEVICE):
    n = 1
    for s in shape:
        n *= s
    dimensions = dims.dimensions(list(shape)) if strides is None else {"shape": list(shape), "strides": strides}
    return ct.Tensor(device, dimensions, Stub(n, datatype))


def i(*shape):
    return t(*shape, datatype="int")


NORM = blocks.norm_descriptor()
CALLS = [
    ("Unrecognized norm", lambda: blocks.norm_descriptor(post="batch")),
    ("Epsilon", lambda: blocks.norm_descriptor(epsilon=-1)),
    ("shapes differ", lambda: blocks.norm_residual(t(4, 8), t(4, 8), None, t(4, 9), None, {}, NORM)),
    ("needs a tensor", lambda: blocks.norm_residual(t(4, 8), None, None, t(4, 8), None, {}, NORM)),
    ("float and double", lambda: blocks.norm_residual(i(4, 8), i(4, 8), None, i(4, 8), None, {}, NORM)),
    ("required datatype", lambda: blocks.norm_residual(t(4, 8), t(4, 8, datatype="double"), None, t(4, 8), None, {}, NORM)),
    ("same device", lambda: blocks.norm_residual(t(4, 8), t(4, 8, device=object()), None, t(4, 8), None, {}, NORM)),
    ("contiguous", lambda: blocks.norm_residual(t(4, 8), t(4, 8), None, t(4, 8, strides=[1, 4]), None, {}, NORM)),
    ("dense tensor of shape", lambda: blocks.norm_residual(t(4, 8), t(4, 8), t(2, 4), t(4, 8), None, {}, NORM)),
    ("dense tensor of shape", lambda: blocks.norm_residual(t(4, 8), t(4, 8), None, t(4, 8), None, {"pre-scale": t(7)}, NORM)),
    ("unknown parameters", lambda: blocks.norm_residual(t(4, 8), t(4, 8), None, t(4, 8), None, {"scale": t(8)}, NORM)),
    ("gate's shape", lambda: blocks.norm_residual(t(4, 8), t(4, 8), None, t(4, 8), None, {"gate": t(2, 8)}, NORM)),
    ("which is no parameter", lambda: blocks.norm_residual_gradient(t(4, 8), None, {"gate": t(1, 8)}, t(4, 8), None, t(4, 8), t(4, 8),
                                                                    t(4, 4), {}, NORM)),
    ("of at most 1024", lambda: blocks.route_experts(i(5, 9), t(5, 9), i(9), i(45), i(5, 9), t(5, 8))),
    ("must be an int", lambda: blocks.route_experts(t(5, 2), t(5, 2), i(9), i(10), i(5, 2), t(5, 8))),
    ("dense tensor of shape", lambda: blocks.route_experts(i(5, 2), t(5, 2), i(8), i(10), i(5, 2), t(5, 8))),
    ("logits are needed", lambda: blocks.route_experts_gradient(t(5, 8), t(5, 2), t(5, 2), i(5, 2), None, renormalize=False)),
    ("do not go together", lambda: blocks.grouped_gemm(t(10, 6), True, 1.0, t(10, 8), t(3, 6, 7), 0.0, i(4))),
    ("matrix to each group", lambda: blocks.grouped_gemm(t(10, 6), True, 1.0, t(10, 8), t(6, 8), 0.0, i(4))),
    ("dense tensor of shape", lambda: blocks.grouped_gemm(t(10, 6), True, 1.0, t(10, 8), t(3, 6, 8), 0.0, i(3))),
    ("A has 9 rows", lambda: blocks.grouped_gemm(t(10, 6), True, 1.0, t(9, 8), t(3, 6, 8), 0.0, i(4))),
    ("dense tensor of shape", lambda: blocks.grouped_gemm(t(10, 6), True, 1.0, t(9, 8), t(3, 6, 8), 0.0, i(4), index=i(9))),
    ("do not go with", lambda: blocks.grouped_gemm_weights(t(3, 6, 8), 1.0, t(10, 6), t(10, 7), 0.0, i(4))),
    ("different numbers of rows", lambda: blocks.grouped_gemm_weights(t(3, 6, 8), 1.0, t(10, 6), t(9, 8), 0.0, i(4))),
    ("rows of 7", lambda: blocks.combine_experts(t(5, 8), t(10, 7), t(5, 2), i(5, 2))),
    ("dense tensor of shape", lambda: blocks.combine_experts(t(5, 8), t(10, 8), t(5, 3), i(5, 2))),
    ("rows are needed", lambda: blocks.combine_experts_gradient(None, t(5, 2), t(5, 8), None, None, i(5, 2))),
    ("does not go with", lambda: blocks.combine_experts_gradient(t(9, 8), t(5, 2), t(5, 8), t(10, 8), None, i(5, 2))),
    ("two values", lambda: optimize.clip_gradients(optimize.Backend(Stub()), [t(4)], 1.0, t(3))),
    ("must be positive", lambda: optimize.clip_gradients(optimize.Backend(Stub()), [t(4)], 0.0, t(2))),
    ("differ in their lengths", lambda: optimize.clip_gradients(optimize.Backend(Stub()), [t(4)], 1.0, t(2), [t(5)])),
    ("must be dense", lambda: optimize.clip_gradients(optimize.Backend(Stub()), [t(4, 4, strides=[8, 1])], 1.0, t(2))),
    ("datatype mismatch", lambda: optimize.clip_gradients(optimize.Backend(Stub()), [t(4, datatype="double")], 1.0, t(2))),
]


@pytest.mark.parametrize("message,call", CALLS, ids=[f"{n} {m}" for n, (m, _) in enumerate(CALLS)])
def test_tensor_api(message, call):
    with ct.tensor_context(Stub(), "float"):
        with pytest.raises((ValueError, TypeError)) as e:
            call()
    assert message in str(e.value), str(e.value)


# ---------------------------------------------------------------- operands found in native code

class Recorder:
    """A stream that notes the calls it gets."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        plain = lambda a: (tuple(a["shape"]), tuple(a["strides"])) if isinstance(a, dict) else a.key if isinstance(a, Keyed) else a
        return lambda *args: self.calls.append((name, [plain(a) for a in args]))


class Keyed(Stub):
    """A buffer that is told apart from others."""


def operand(rng, shape, datatype, key):
    """A tensor of this shape, or of one near it, in rows that may lie apart; now and then of another type, or none."""
    shape = list(shape)
    if rng.random() < 0.06:
        shape[rng.randrange(len(shape))] += rng.choice([-1, 1, 3])
    if rng.random() < 0.04:
        shape = rng.choice([[1] + shape, shape[1:] or [1], shape + [1], [0] + shape[1:]])
    if rng.random() < 0.04:
        return None
    if rng.random() < 0.05:
        datatype = rng.choice(["float", "double", "int", "byte"])
    strides = dims.dimensions(shape)["strides"] if all(shape) else [1] * len(shape)
    if len(shape) > 1 and rng.random() < 0.3:
        pad = rng.choice([1, 5, -1])
        strides = [s + pad for s in strides[:-1]] + strides[-1:]
    if rng.random() < 0.04:
        strides = strides[:-1] + [2]
    n = 1
    for s in shape:
        n *= s
    buffer = Keyed(n, datatype)
    buffer.key = (key, datatype)
    return ct.Tensor(DEVICE if rng.random() < 0.97 else "another", {"shape": shape, "strides": strides}, buffer)


def drawn_call(rng):
    n, width, experts, chosen = rng.randint(1, 4), rng.randint(1, 5), rng.randint(1, 4), rng.randint(1, 3)
    columns, rows, real = rng.randint(1, 5), rng.randint(1, 6), rng.choice(["float", "double"])
    count = iter(range(100))
    f, j = (lambda *s: operand(rng, s, real, next(count))), (lambda *s: operand(rng, s, "int", next(count)))
    maybe = lambda x: x if rng.random() < 0.7 else None
    kind = rng.randrange(7)
    if kind < 2:
        d = blocks.norm_descriptor(post=rng.choice(blocks.NORM_KINDS), pre=rng.choice(blocks.NORM_KINDS))
        p = {k: maybe(f(width)) for k in ("post-scale", "post-bias", "pre-scale", "pre-bias")}
        p["gate"] = maybe(f(rng.choice([1, n]), rng.choice([1, width])))
        if kind == 0:
            args = f(n, width), f(n, width), maybe(f(4, n)), f(n, width), maybe(f(n, width)), p, d
            return lambda: blocks.norm_residual(*args)
        g = {k: maybe(f(*t.shape())) for k, t in p.items() if t is not None and all(s >= 0 for s in t.shape())}
        args = f(n, width), maybe(f(n, width)), g, maybe(f(n, width)), maybe(f(n, width)), f(n, width), f(n, width), f(4, n), p, d
        return lambda: blocks.norm_residual_gradient(*args)
    if kind == 2:
        args = j(n, chosen), f(n, chosen), j(experts + 1), j(n * chosen), j(n, chosen), f(n, experts)
        return lambda: blocks.route_experts(*args)
    if kind == 3:
        args, renormalize = (f(n, experts), f(n, chosen), f(n, chosen), j(n, chosen), maybe(f(n, experts))), rng.random() < 0.5
        return lambda: blocks.route_experts_gradient(*args, renormalize=renormalize)
    if kind == 4:
        trans, index = rng.random() < 0.5, maybe(j(rows))
        args = (f(rows, columns), trans, 1.0, f(rows if index is None else n, width), f(experts, *((columns, width) if trans else (width, columns))),
                0.0, j(experts + 1))
        return lambda: blocks.grouped_gemm(*args, index=index)
    if kind == 5:
        ia, ib = maybe(j(rows)), maybe(j(rows))
        args = f(experts, width, columns), 1.0, f(rows if ia is None else n, width), f(rows if ib is None else n + 1, columns), 0.0, j(experts + 1), ia, ib
        return lambda: blocks.grouped_gemm_weights(*args)
    if rng.random() < 0.5:
        args = f(n, width), f(rows, width), maybe(f(n, chosen)), j(n, chosen)
        return lambda: blocks.combine_experts(*args)
    args = maybe(f(rows, width)), maybe(f(n, chosen)), f(n, width), maybe(f(rows, width)), maybe(f(n, chosen)), j(n, chosen)
    return lambda: blocks.combine_experts_gradient(*args)


@pytest.mark.skipif(capi.front is None, reason="the native front is not built")
def test_native_operands_are_those_of_the_checks(monkeypatch):
    """Calls drawn with operands that fit, or nearly: with the operands found in native code and without, the same call
    reaches the stream, or the same error is raised."""
    import random
    reached = refused = 0
    for seed in range(8000):
        outcomes = []
        for native in (True, False):
            with monkeypatch.context() as m:
                if not native:
                    m.setattr(blocks, "_operands", lambda kinds, tensors: None)
                stream = Recorder()
                call = drawn_call(random.Random(seed))
                with ct.tensor_context(stream, "float"):
                    try:
                        call()
                        outcomes.append(stream.calls)
                    except (ValueError, TypeError) as e:
                        assert not stream.calls
                        outcomes.append((type(e), str(e)))
        assert outcomes[0] == outcomes[1], seed
        reached += isinstance(outcomes[0], list)
        refused += not isinstance(outcomes[0], list)
    assert reached > 1000 and refused > 1000, (reached, refused)
