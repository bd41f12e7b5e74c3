"""What the gated products refuse, checked on the host ahead of any device call.  Nothing here needs a GPU."""
import numpy as np
import pytest

from cortex_amd import blocks
from cortex_amd import capi
from cortex_amd import tensor as ct
from test_orthogonalize_refusals import A, Device, matrix, refuses

F = capi.F32


def gated(**change):
    args = dict(stream=None, inner=A[0], inner_colstride=12, pre=A[1], pre_colstride=24, activation=3, a=A[2], a_row_count=30, a_col_count=16,
                a_colstride=16, index=A[3], b=A[4], hidden=12, b_colstride=16, b_stride=384, offsets=A[5], n_groups=3, row_count=20, dtype=F)
    args.update(change)
    return list(args.values())


@pytest.mark.parametrize("message,change", [
    ("float or double", {"dtype": capi.I32}), ("unknown activation", {"activation": 5}), ("unknown activation", {"activation": -1}),
    ("bad extent", {"a_row_count": -1}), ("bad extent", {"hidden": 1 << 30}), ("bad extent", {"row_count": 1 << 31}), ("bad extent", {"hidden": 1 << 62}),
    ("groups, at most", {"n_groups": 65536}), ("without offsets", {"offsets": None}), ("null buffer", {"inner": None}), ("null buffer", {"a": None}),
    ("null buffer", {"b": None}), ("rows of", {"index": None, "a_row_count": 19}), ("column stride", {"inner_colstride": 11}),
    ("column stride", {"pre_colstride": 23}), ("column stride", {"a_colstride": 15}), ("column stride", {"b_colstride": 15}),
    ("negative stride", {"b_stride": -1}), ("beyond 2^40", {"b_stride": 1 << 41}), ("results overlap", {"pre": A[0] + 4}),
    ("overlaps an operand", {"inner": A[2]}), ("overlaps an operand", {"pre": A[2] + 64}), ("overlaps an operand", {"inner": A[4] + 1000}),
    ("offsets or the index", {"inner": A[5]}), ("offsets or the index", {"pre": A[3]})], ids=str)
def test_gated_gemm(message, change):
    refuses(message, "ct_gated_gemm", *gated(**change))


def gradient(**change):
    args = dict(stream=None, pre_gradient=A[0], pre_gradient_colstride=24, inner=A[1], inner_colstride=12, activation=4, a=A[2], a_col_count=16,
                a_colstride=16, b=A[3], hidden=12, b_colstride=12, b_stride=192, pre=A[4], pre_colstride=24, offsets=A[5], n_groups=3, row_count=20,
                dtype=F)
    args.update(change)
    return list(args.values())


@pytest.mark.parametrize("message,change", [
    ("float or double", {"dtype": capi.I8}), ("unknown activation", {"activation": 9}), ("bad extent", {"a_col_count": -1}), ("bad extent", {"hidden": 1 << 30}),
    ("groups, at most", {"n_groups": -1}), ("without offsets", {"offsets": None}), ("null buffer", {"pre": None}), ("null buffer", {"pre_gradient": None}),
    ("null buffer", {"a": None}), ("null buffer", {"b": None}), ("column stride", {"pre_gradient_colstride": 23}), ("column stride", {"inner_colstride": 11}),
    ("column stride", {"a_colstride": 15}), ("column stride", {"b_colstride": 11}), ("column stride", {"pre_colstride": 20}),
    ("negative stride", {"b_stride": -1}), ("beyond 2^40", {"a_colstride": 1 << 41}), ("results overlap", {"inner": A[0] + 8}),
    ("overlaps pre", {"pre_gradient": A[4] + 4}), ("overlaps pre", {"pre_gradient": A[4], "pre_gradient_colstride": 25}), ("overlaps pre", {"inner": A[4]}),
    ("overlaps an operand", {"pre_gradient": A[2]}), ("overlaps an operand", {"inner": A[3]}), ("overlaps the offsets", {"inner": A[5]})], ids=str)
def test_gated_gemm_gradient(message, change):
    refuses(message, "ct_gated_gemm_gradient", *gradient(**change))


M, I = matrix, lambda n: matrix(n, datatype="int")


@pytest.mark.parametrize("message,args,kwargs", [
    ("unrecognized activation", (M(4, 6), None, M(4, 5), M(12, 5)), {"activation": "softplus"}), ("is needed", (M(4, 6), None, None, M(12, 5)), {}),
    ("float and double", (I(4), None, M(4, 5), M(12, 5)), {}), ("required datatype", (M(4, 6), None, M(4, 5), M(12, 5, datatype="double")), {}),
    ("do not go together", (M(4, 6), None, M(4, 5), M(11, 5)), {}), ("do not go together", (M(4, 6), None, M(4, 5), M(12, 6)), {}),
    ("pre must be", (M(4, 6), M(4, 11), M(4, 5), M(12, 5)), {}), ("must be a matrix", (M(4, 6), None, M(4, 5), M(2, 12, 5)), {}),
    ("matrix to each group", (M(4, 6), None, M(4, 5), M(12, 5), I(2)), {}), ("offsets must be", (M(4, 6), None, M(4, 5), M(2, 12, 5), I(2)), {}),
    ("index must be", (M(4, 6), None, M(9, 5), M(12, 5), None, I(5)), {}), ("A has 9 rows", (M(4, 6), None, M(9, 5), M(12, 5)), {}),
    ("contiguous", (M(4, 6, strides=[1, 4]), None, M(4, 5), M(12, 5)), {}), ("same device", (M(4, 6), None, M(4, 5, device=Device()), M(12, 5)), {})], ids=str)
def test_tensors(message, args, kwargs):
    with pytest.raises(ct.TensorError, match=message):
        blocks.gated_gemm(*args, **kwargs)


@pytest.mark.parametrize("message,args,kwargs", [
    ("unrecognized activation", (M(4, 12), None, M(4, 5), M(5, 6), M(4, 12)), {"activation": None}), ("is needed", (M(4, 12), None, M(4, 5), M(5, 6), None), {}),
    ("do not go together", (M(4, 12), None, M(4, 5), M(6, 6), M(4, 12)), {}), ("pre and its gradient", (M(4, 12), None, M(3, 5), M(5, 6), M(4, 12)), {}),
    ("pre and its gradient", (M(4, 12), None, M(4, 5), M(5, 6), M(4, 11)), {}), ("inner must be", (M(4, 12), M(4, 5), M(4, 5), M(5, 6), M(4, 12)), {}),
    ("offsets must be", (M(4, 12), None, M(4, 5), M(2, 5, 6), M(4, 12), I(4)), {}), ("required datatype", (M(4, 12), None, M(4, 5), M(5, 6), M(4, 12, datatype="double")), {})], ids=str)
def test_tensors_of_the_gradient(message, args, kwargs):
    with pytest.raises(ct.TensorError, match=message):
        blocks.gated_gemm_gradient(*args, **kwargs)


def test_layers():
    with pytest.raises(ct.TensorError, match="unrecognized activation"):
        blocks.GatedBlock(4, 8, 8, activation="none")
    with pytest.raises(ct.TensorError, match="unrecognized activation"):
        blocks.ExpertBlock(4, 8, 8, 2, 1, gated="none")
