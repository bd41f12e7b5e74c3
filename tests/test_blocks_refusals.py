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
