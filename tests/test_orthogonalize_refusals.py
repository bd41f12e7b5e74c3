"""What the orthogonalisation and the optimizer step made of it refuse, checked on the host ahead of any device call; and what
the workspace is.  Nothing here needs a GPU."""
import array
import ctypes as C

import numpy as np
import pytest

from cortex_amd import capi
from cortex_amd import optimize
from cortex_amd import tensor as ct

A = [0x10000000 * (i + 1) for i in range(8)]     # addresses that nothing follows
TRIPLES = array.array("d", optimize.NEWTON_SCHULZ_COEFFICIENTS * 5).tobytes()
ROOM = 1 << 24


def refuses(message, name, *args):
    with pytest.raises(capi.CortexHipError) as e:
        capi.call(name, *args)
    assert e.value.status == 1 and message in e.value.message, e.value.message


def orthogonalize(**change):
    args = dict(stream=None, output=A[0], output_colstride=40, output_stride=1200, alpha=1.0, input=A[1], input_colstride=40, input_stride=1200,
                beta=0.0, count=2, rows=30, columns=40, coefficients=TRIPLES, steps=5, epsilon=1e-7, workspace=A[2], workspace_bytes=ROOM,
                dtype=capi.F32)
    args.update(change)
    return list(args.values())


def of(*values):
    return array.array("d", values).tobytes()


@pytest.mark.parametrize("message,change", [
    ("float or double", {"dtype": capi.I32}), ("negative extent", {"count": -1}), ("negative extent", {"rows": -1}), ("a side are taken", {"rows": (1 << 21) + 1}),
    ("a side are taken", {"count": 65536}), ("elements are taken", {"rows": 1 << 16, "columns": 1 << 15, "output_colstride": 1 << 15, "count": 1, "input_colstride": 1 << 15}),
    ("steps", {"steps": 0}), ("steps", {"steps": 65}), ("null coefficients", {"coefficients": None}), ("epsilon", {"epsilon": -1e-9}),
    ("epsilon", {"epsilon": float("nan")}), ("null buffer", {"output": None}), ("null buffer", {"input": None}), ("workspace must be", {"workspace": None}),
    ("aligned to 16", {"workspace": A[2] + 8}), ("a matrix takes", {"workspace_bytes": 1000}), ("a matrix takes", {"workspace_bytes": -1}),
    ("below the row's length", {"output_colstride": 39}), ("below the row's length", {"input_colstride": 39}), ("negative stride", {"input_stride": -1}),
    ("results overlap", {"output_stride": 1199}), ("overlaps the input", {"output": A[1] + 4}), ("overlaps the input", {"output": A[1], "output_stride": 1300}),
    ("workspace overlaps", {"workspace": A[1] + 16}), ("workspace overlaps", {"workspace": A[0]}), ("workspace overlaps", {"workspace": A[0] - ROOM + 16}),
    ("finite", {"coefficients": of(1.0, float("nan"), 0.0), "steps": 1}), ("finite", {"coefficients": of(float("inf"), 0.0, 0.0), "steps": 1}),
    ("beyond 2^40", {"coefficients": of(2.0 ** 41, 0.0, 0.0), "steps": 1}), ("beyond 2^40", {"coefficients": of(*[32.0, 0.0, 0.0] * 9), "steps": 9})], ids=str)
def test_orthogonalize(message, change):
    refuses(message, "ct_orthogonalize", *orthogonalize(**change))


@pytest.mark.parametrize("coefficients", [(2.0 ** 31, 0.0, 0.0, 1.0, 0.0, 0.0), (2.0 ** 33, 0.0, 0.0, 0.5, 0.0, 0.0, 2.0, 0.0, 0.0)], ids=str)
def test_singular_values_whose_fourth_power_is_no_float(coefficients):
    """A A of a singular value of 2^33 is 2^132, which a float does not hold; as the last step's result that value may be."""
    change = {"coefficients": of(*coefficients), "steps": len(coefficients) // 3}
    refuses("beyond 2^30 before the last step", "ct_orthogonalize", *orthogonalize(**change))
    refuses("beyond 2^30 before the last step", "ct_muon_step", *step(**change))
    for allowed in (orthogonalize(coefficients=of(*coefficients), steps=1, workspace=None), orthogonalize(dtype=capi.F64, workspace=None, **change)):
        refuses("workspace must be", "ct_orthogonalize", *allowed)


def step(**change):
    args = dict(stream=None, dtype=capi.F32, alpha=0.02, momentum=0.95, nesterov=1, weight_decay=0.0, gradient_alpha=1.0, coefficients=TRIPLES, steps=5,
                epsilon=1e-7, gradient=A[0], parameters=A[1], momentum_vals=A[2], count=2, rows=30, columns=40, workspace=A[3], workspace_bytes=ROOM)
    args.update(change)
    return list(args.values())


@pytest.mark.parametrize("message,change", [
    ("float or double", {"dtype": capi.I64}), ("negative extent", {"columns": -3}), ("null buffer", {"gradient": None}), ("null buffer", {"parameters": None}),
    ("null buffer", {"momentum_vals": None}), ("overlap", {"gradient": A[1]}), ("overlap", {"momentum_vals": A[0] + 400}), ("overlap", {"parameters": A[2]}),
    ("workspace overlaps", {"workspace": A[2]}), ("workspace overlaps", {"workspace": A[0] + 16}), ("workspace overlaps", {"workspace": A[1] + 16}),
    ("steps", {"steps": -1}), ("workspace must be", {"workspace": None})], ids=str)
def test_step(message, change):
    refuses(message, "ct_muon_step", *step(**change))


def workspace(count, rows, columns, dtype=capi.F32):
    need = C.c_int64(-1)
    capi.call("ct_orthogonalize_workspace", count, rows, columns, dtype, C.byref(need))
    return need.value


def test_workspace():
    assert workspace(0, 3, 4) == workspace(2, 0, 4) == 0
    one = workspace(1, 100, 300)
    assert workspace(7, 100, 300) == 7 * one and workspace(1, 300, 100) == one
    # beyond what fills the chip matrices take turns
    assert workspace(1000, 1024, 1024) == 64 * workspace(1, 1024, 1024)
    # three float matrices in two pieces, two of the shorter side; three in double there are two
    assert 12 * 1024 * 2048 + 8 * 1024 * 1024 <= workspace(1, 1024, 2048) <= 12 * 1024 * 2048 + 8 * 1024 * 1024 + (1 << 16)
    # rows of doubles are an odd number of 128 bytes apart: up to 31 doubles more to each of four times 1024 rows
    assert 16 * 1024 * 2048 + 16 * 1024 * 1024 <= workspace(1, 1024, 2048, capi.F64) <= 16 * 1024 * 2048 + 16 * 1024 * 1024 + 4 * 1024 * 31 * 8 + (1 << 16)
    refuses("float or double", "ct_orthogonalize_workspace", 1, 2, 3, capi.I8, C.byref(C.c_int64()))
    refuses("null result", "ct_orthogonalize_workspace", 1, 2, 3, capi.F32, None)
    refuses("bad extent", "ct_orthogonalize_workspace", 1, 1 << 22, 3, capi.F32, C.byref(C.c_int64()))


class Device:
    pass


class Buffer:
    def __init__(self, n, datatype="float", device=None):
        self.n, self.datatype, self.device, self.ptr = n, datatype, device or DEVICE, A[0]

    def ecount(self):
        return self.n

    def get_datatype(self):
        return self.datatype

    def sub_buffer(self, offset, n):
        assert offset + n <= self.n
        return Buffer(n, self.datatype, self.device)


DEVICE = Device()


def matrix(*shape, strides=None, datatype="float", device=None):
    return ct.Tensor(device or DEVICE, {"shape": list(shape), "strides": strides or [int(np.prod(shape[i + 1:])) for i in range(len(shape))]},
                     Buffer(int(np.prod(shape)), datatype, device))


@pytest.mark.parametrize("error,message,output,input,kwargs", [
    (ValueError, "must be a tensor", Buffer(12), matrix(3, 4), {}), (ValueError, "must be a matrix", matrix(12), matrix(12), {}),
    (ValueError, "differ", matrix(3, 4), matrix(4, 3), {}), (ValueError, "contiguous", matrix(3, 4, strides=[1, 3]), matrix(3, 4), {}),
    (ValueError, "contiguous", matrix(3, 4), matrix(3, 4, strides=[3, 1]), {}), (TypeError, "datatype", matrix(3, 4, datatype="double"), matrix(3, 4), {}),
    (ValueError, "same device", matrix(3, 4, device=Device()), matrix(3, 4), {}), (ValueError, "three numbers", matrix(3, 4), matrix(3, 4), {"coefficients": (1.0, 2.0)}),
    (ValueError, "none", matrix(3, 4), matrix(3, 4), {"coefficients": ()}),
    (ValueError, "three numbers", matrix(3, 4), matrix(3, 4), {"coefficients": [(1.0, 2.0, 3.0)] * 4})], ids=str)
def test_tensors(error, message, output, input, kwargs):
    with pytest.raises(error, match=message):
        optimize.orthogonalize(optimize.Backend(None, "float"), output, input, workspace=Buffer(1 << 20, "byte"), **kwargs)


@pytest.mark.parametrize("error,message,gradient,parameters,momentum", [
    (ValueError, "must be a tensor", matrix(3, 4), Buffer(12), Buffer(12)), (ValueError, "must be a matrix", matrix(12), matrix(12), Buffer(12)),
    (ValueError, "dense", matrix(3, 4), matrix(3, 4, strides=[5, 1]), Buffer(12)), (ValueError, "dense", matrix(4, 3), matrix(3, 4), Buffer(12)),
    (TypeError, "datatype", matrix(3, 4, datatype="double"), matrix(3, 4), Buffer(12)), (ValueError, "a gradient of 11", Buffer(11), matrix(3, 4), Buffer(12)),
    (ValueError, "same device", matrix(3, 4, device=Device()), matrix(3, 4), Buffer(12))], ids=str)
def test_optimizer(error, message, gradient, parameters, momentum):
    optimizer = optimize.create_optimizer(optimize.Backend(None, "float"), optimize.muon())
    with pytest.raises(error, match=message):
        optimizer.compute_parameters({"momentum-vals": momentum}, 1.0, 0, gradient, parameters)
    with pytest.raises(TypeError):
        optimize.create_optimizer(optimize.Backend(None, "int"), optimize.muon())


def test_a_workspace_of_another_device():
    with pytest.raises(ValueError, match="same device"):
        optimize.orthogonalize(optimize.Backend(None, "float"), matrix(3, 4), matrix(3, 4), workspace=Buffer(1 << 20, "byte", Device()))
