"""Calls of the operators of residual blocks with experts that are refused, or that reach the stream, by how their operands lie
in memory.  Nothing here needs a GPU."""
import ctypes as C
import random
import struct

import numpy as np
import pytest

from cortex_amd import blocks
from cortex_amd import capi
from cortex_amd import optimize
from cortex_amd import tensor as ct
from test_blocks_refusals import A, Recorder, combine, combine_gradient, d, grouped, norm, norm_gradient, refuses, route, route_gradient, t, weights


# ---------------------------------------------------------------- clipping: the order of elements

def at(ptr, *shape, strides=None, count=None):
    """A float tensor of which the memory begins at an address."""
    x = t(*shape, strides=strides)
    x.buffer.ptr = ptr
    if count is not None:
        x.buffer._ecount = count
    return x


class Buffer:
    """A buffer and nothing else: no tensor."""

    def __init__(self, ptr, n):
        self.ptr, self._ecount, self.datatype = ptr, n, "float"

    def ecount(self):
        return self._ecount

    def get_datatype(self):
        return self.datatype


def clipped(gradients, outputs=None, **more):
    """(addresses, addresses of the results) as they reach the stream."""
    stream = Recorder()
    optimize.clip_gradients(optimize.Backend(stream, "float"), gradients, 1.0, at(64, 2), outputs, **more)
    (name, (into_at, counts, into, limit, _)), = stream.calls
    assert name == "clip_gradients"
    unpack = lambda b: None if b is None else struct.unpack(f"{len(b) // 8}q", b)
    return unpack(into_at), unpack(counts), unpack(into)


@pytest.mark.parametrize("native", [True, False])
def test_clipping_takes_results_in_the_order_of_their_gradients(native, monkeypatch):
    if not native:
        monkeypatch.setattr(capi, "front", None)
    elif capi.front is None:
        pytest.skip("the native front is not built")
    plain, turned = at(4096, 2, 3), at(8192, 2, 3, strides=[1, 2])
    # in place every element stays where it is, whatever the order; so it does where both have the same
    assert clipped([turned, plain]) == ((8192, 4096), (6, 6), (8192, 4096))
    assert clipped([turned], in_place=False) == ((8192,), (6,), None)
    assert clipped([turned], [at(12288, 2, 3, strides=[1, 2])]) == ((8192,), (6,), (12288,))
    assert clipped([at(4096, 2, 1, 3, strides=[1, 9, 2])], [at(12288, 2, 3, strides=[1, 2])]) == ((4096,), (6,), (12288,))
    assert clipped([plain], [at(12288, 6)]) == ((4096,), (6,), (12288,))
    assert clipped([at(4096, 0, 5, strides=[1, 1]), plain]) == ((4096, 4096), (0, 6), (4096, 4096))
    assert clipped([plain], [Buffer(12288, 6)]) == ((4096,), (6,), (12288,))
    for gradients, outputs in (([turned], [at(12288, 2, 3)]), ([plain], [at(12288, 2, 3, strides=[1, 2])]), ([turned], [at(12288, 6)]), ([turned], [Buffer(12288, 6)]),
                               ([plain, turned], [turned, plain]), ([at(4096, 3, 2, strides=[1, 3])], [at(12288, 2, 3, strides=[1, 2])])):
        with pytest.raises(ValueError, match="order"):
            clipped(gradients, outputs)


@pytest.mark.parametrize("native", [True, False])
def test_clipping_takes_extents_of_any_whole_number(native, monkeypatch):
    """A shape of numpy's numbers, as other calls take it; an index tensor in its place is refused."""
    if not native:
        monkeypatch.setattr(capi, "front", None)
    x, turned = at(4096, 2, 3), at(8192, 2, 3)
    x.dimensions = {"shape": [np.int64(2), np.int32(3)], "strides": [np.int64(3), 1]}
    turned.dimensions = {"shape": [np.int64(2), 3], "strides": [1, np.int64(2)]}
    assert clipped([x, turned]) == ((4096, 8192), (6, 6), (4096, 8192))
    assert clipped([x], [at(12288, 6)]) == ((4096,), (6,), (12288,))
    with pytest.raises(ValueError, match="order"):
        clipped([turned], [at(12288, 6)])
    indexed = at(4096, 2, 3, count=100)
    indexed.dimensions = {"shape": [t(2, datatype="int"), 3], "strides": [3, 1]}
    with pytest.raises(ValueError, match="must be dense"):
        clipped([indexed])


@pytest.mark.parametrize("native", [True, False])
def test_clipping_takes_tensors_that_fill_their_memory(native, monkeypatch):
    """A row that is given again and again, or rows apart: what lies between is no gradient."""
    if not native:
        monkeypatch.setattr(capi, "front", None)
    for shape, strides in (([4, 4], [4, 0]), ([4, 4], [8, 1]), ([2, 3], [3, 2])):
        with pytest.raises(ValueError, match="must be dense"):
            clipped([at(4096, *shape, strides=strides, count=100)])


# ---------------------------------------------------------------- overlaps
#
# Every operand is at an address of its own, 1 MiB from the next one (test_blocks_refusals).  What is moved here meets another
# one's elements in one place at least: the call would read what it has stored, or store twice to one place.

LAST = 4 * (4 * 8 - 1)      # bytes from the first element of 4 rows of 8 floats to their last


@pytest.mark.parametrize("change", [
    {"statistics": A[3]}, {"statistics": A[3] + LAST}, {"statistics": A[4] - 4 * 15}, {"statistics": A[5] + 28}, {"statistics": A[6] + 28},
    {"statistics": A[7] - 60}, {"post_bias": A[2] + 60}, {"pre_bias": A[2] - 28}], ids=str)
def test_norm_statistics_that_overlap(change):
    refuses("the statistics overlap an operand", "ct_norm_residual", *norm(**change))


@pytest.mark.parametrize("message,change", [
    ("scale or bias overlaps", {"post_scale_gradient": A[11]}), ("scale or bias overlaps", {"post_scale_gradient": A[7] + LAST}),
    ("scale or bias overlaps", {"post_bias_gradient": A[5]}), ("scale or bias overlaps", {"post_bias_gradient": A[6] - 28}),
    ("scale or bias overlaps", {"pre_scale_gradient": A[12]}), ("scale or bias overlaps", {"pre_bias_gradient": A[8] + 4}),
    ("scale or bias overlaps", {"pre_scale_gradient": A[9] + 60}), ("scale or bias overlaps", {"pre_bias_gradient": A[10]}),
    ("gate's gradient overlaps", {"gate_gradient": A[9] + 60}), ("gate's gradient overlaps", {"gate_gradient": A[11] - 28}),
    ("results overlap", {"post_bias_gradient": A[3] + 28}), ("results overlap", {"pre_bias_gradient": A[4] - 28}),
    ("results overlap", {"gate_gradient": A[3]}), ("results overlap", {"pre_scale_gradient": A[3]}),
    ("overlaps an operand", {"pre_scale_gradient": A[0] + LAST}), ("overlaps an operand", {"gate_gradient": A[1] - 28})], ids=str)
def test_norm_gradients_that_overlap(message, change):
    refuses(message, "ct_norm_residual_gradient", *norm_gradient(**change))


@pytest.mark.parametrize("change", [{"post_scale_gradient": A[7] + 4 * 57}, {"pre_scale_gradient": A[8] + 4 * 7},
                                    {"gate_gradient": A[7] + 4 * (3 * 64 - 7)}], ids=str)
def test_vectors_that_reach_from_a_gap_into_a_row(change):
    apart = d(4, 8, strides=[64, 1])
    refuses("overlaps an operand", "ct_norm_residual_gradient", *norm_gradient(input_dims=apart, output_dims=apart, **change))


@pytest.mark.parametrize("message,change", [
    ("results overlap", {"weights": A[0] + 4 * 39}), ("results overlap", {"offsets": A[0] - 4 * 16}), ("results overlap", {"tokens": A[2] + 4 * 16}),
    ("results overlap", {"slots": A[3]}), ("results overlap", {"slots": A[1] + 8 * 39, "dtype": capi.F64}),
    ("the logits", {"experts": A[5] + 4 * 159}), ("the logits", {"weights": A[5]}), ("the logits", {"offsets": A[5] - 4 * 16}),
    ("the logits", {"tokens": A[5] + 4 * 32}), ("the logits", {"slots": A[5] + 4 * (9 * 40 + 15), "logits_colstride": 40})], ids=str)
def test_routing_into_what_overlaps(message, change):
    refuses(message, "ct_route_experts", *route(**change))


@pytest.mark.parametrize("change", [
    {"weights_gradient": A[0]}, {"weights": A[0] + 4 * 159}, {"experts": A[0] - 4 * 39}, {"logits": A[0] + 4},
    {"logits": A[0], "logits_colstride": 17}, {"weights": A[0] + 4 * 159, "renormalize": 1},
    {"weights": A[0] + 4 * 17, "logits_gradient_colstride": 60, "n_chosen": 5}], ids=str)
def test_routing_gradients_that_overlap(change):
    refuses("overlaps an operand", "ct_route_experts_gradient", *route_gradient(**change))


@pytest.mark.parametrize("message,change", [
    ("weights or the slots", {"weights": A[0] + 4 * 79}), ("weights or the slots", {"weights": A[0] - 4 * 19}), ("weights or the slots", {"slots": A[0]}),
    ("weights or the slots", {"slots": A[0] + 4 * (9 * 30 + 7), "output_colstride": 30}),
    ("weights or the slots", {"weights": A[0] - 8 * 19, "dtype": capi.F64})], ids=str)
def test_combining_into_what_overlaps(message, change):
    refuses(message, "ct_combine_experts", *combine(**change))


@pytest.mark.parametrize("message,change", [
    ("rows_gradient overlaps", {"weights": A[0] + 4 * 159}), ("rows_gradient overlaps", {"slots": A[0] - 4 * 19}),
    ("weights_gradient overlaps", {"weights_gradient": A[2]}), ("weights_gradient overlaps", {"weights_gradient": A[3] + 4 * 159}),
    ("weights_gradient overlaps", {"weights_gradient": A[5] + 4 * 19}), ("weights_gradient overlaps", {"weights_gradient": A[4] + 4}),
    ("weights_gradient overlaps", {"weights_gradient": A[4] - 4 * 19}), ("results overlap", {"weights_gradient": A[0] + 4 * 159}),
    ("weights_gradient overlaps", {"weights_gradient": A[5], "rows_gradient": None})], ids=str)
def test_combining_gradients_that_overlap(message, change):
    refuses(message, "ct_combine_experts_gradient", *combine_gradient(**change))


@pytest.mark.parametrize("change", [{"offsets": A[0] + 4 * 639}, {"offsets": A[0] - 4 * 3}, {"index": A[0] - 4 * 19}, {"index": A[0] + 4 * 320},
                                    {"index": A[0] + 8 * 90 * 3 - 4 * 19, "c_colstride": 90, "dtype": capi.F64}], ids=str)
def test_products_into_their_offsets_or_index(change):
    refuses("offsets or the index", "ct_grouped_gemm", *grouped(**change))


@pytest.mark.parametrize("change", [{"offsets": A[0] + 4 * 1535}, {"offsets": A[0] - 4 * 3}, {"a_index": A[0] - 4 * 19}, {"b_index": A[0] + 4 * 512}], ids=str)
def test_products_over_rows_into_their_offsets_or_indexes(change):
    refuses("offsets or an index", "ct_grouped_gemm_weights", *weights(**change))


# ---------------------------------------------------------------- clipping: outputs and other tensors

def clip(gradients, outputs, counts, result=A[20], dtype=capi.F32):
    n = len(gradients)
    addresses = lambda x: None if x is None else (C.c_void_p * n)(*x)
    return None, addresses(gradients), addresses(outputs), (C.c_int64 * n)(*counts), n, 1.0, result, dtype


@pytest.mark.parametrize("message,gradients,outputs,counts", [
    ("overlaps another", [A[0], A[1]], [A[1], A[2]], [8, 8]), ("overlaps another", [A[0], A[1]], [A[2], A[0] + 28], [8, 8]),
    ("overlaps another", [A[0], A[1]], [A[1] - 28, A[1]], [8, 8]), ("overlaps another", [A[0], A[1]], [A[2], A[2] + 28], [8, 8]),
    ("overlaps another", [A[0], A[0]], [A[0], A[0]], [8, 8]), ("overlaps another", [A[0], A[1]], [A[1], A[0]], [8, 8]),
    ("overlaps another", [A[0], A[5], A[1]], [A[0], A[1] - 4 * 7, A[1]], [8, 8, 8]),
    ("norm and the factor overlap tensor 1", [A[0], A[20] - 28], None, [8, 8]), ("norm and the factor overlap tensor 0", [A[0], A[1]], [A[20] + 4, A[2]], [8, 8])])
def test_clipping_into_another_tensor(message, gradients, outputs, counts):
    refuses(message, "ct_clip_gradients", *clip(gradients, outputs, counts))


def test_clipping_long_lists_into_another_tensor():
    """Lists drawn at random, in any order, whose tensors touch but do not meet, but for one output: that one is named, or the tensor
    that it meets."""
    for seed in range(200):
        rng = random.Random(seed)
        n = rng.choice([2, 3, 50, 119, 120, 121, 300])
        counts = [rng.randint(0, 9) for _ in range(n)]
        places, at = {}, 1 << 20
        for slot in rng.sample(range(2 * n), 2 * n):
            places[slot] = at
            at += 4 * counts[slot % n]
        gradients = [places[i] for i in range(n)]
        outputs = [g if rng.random() < 0.5 else places[n + i] for i, g in enumerate(gradients)]
        some = [i for i in range(n) if counts[i]]
        if len(some) < 2:
            continue
        i, j = rng.sample(some, 2)
        meets = rng.choice([gradients[j], outputs[j]])
        # from its last byte before the other's end to its first after the other's beginning
        outputs[i] = meets + 4 * rng.randint(1 - counts[i], counts[j] - 1)
        with pytest.raises(capi.CortexHipError) as e:
            capi.call("ct_clip_gradients", *clip(gradients, outputs, counts, result=1 << 30))
        assert e.value.status == 1 and "overlaps" in e.value.message, (seed, e.value.message)


@pytest.mark.parametrize("change", [dict(n_groups=65535, row_count=(1 << 31) - 1, a_row_count=(1 << 31) - 1, b_col_count=1 << 20, c_colstride=1 << 20),
                                    dict(row_count=(1 << 31) - 1, a_row_count=(1 << 31) - 1, b_col_count=1 << 20, c_colstride=1 << 20, dtype=capi.F64)], ids=str)
def test_products_of_more_tiles_than_can_be_counted(change):
    far = 1 << 61
    refuses("rows of", "ct_grouped_gemm", *grouped(**{**change, "c": 1 << 62, "a": 1 << 30, "b": far, "offsets": 1 << 20}))


def test_products_over_rows_of_more_tiles_than_can_be_counted():
    side = 1 << 22
    refuses("by 4194304 results", "ct_grouped_gemm_weights",
            *weights(c=1 << 62, c_colstride=side, c_stride=side * side, a=1 << 40, a_col_count=side, a_colstride=side, b=1 << 41, b_col_count=side,
                     b_colstride=side))


# ---------------------------------------------------------------- extents

def whole(*shape, datatype="float"):
    """A tensor whose extents and strides are numpy's whole numbers."""
    x = t(*shape, datatype=datatype)
    x.dimensions = {k: [np.int64(n) for n in x.dimensions[k]] for k in ("shape", "strides")}
    return x


def test_extents_of_any_whole_number():
    """Every call reaches the stream with the numbers that plain ints give."""
    d = blocks.norm_descriptor()
    calls = []
    for f, i in ((t, lambda *s: t(*s, datatype="int")), (whole, lambda *s: whole(*s, datatype="int"))):
        stream = Recorder()
        with ct.tensor_context(stream, "float"):
            p = {"post-scale": f(8), "pre-scale": f(8), "gate": f(4, 1)}
            blocks.norm_residual(f(4, 8), f(4, 8), f(4, 4), f(4, 8), f(4, 8), p, d)
            blocks.norm_residual_gradient(f(4, 8), f(4, 8), {"gate": f(4, 1), "pre-scale": f(8)}, f(4, 8), f(4, 8), f(4, 8), f(4, 8), f(4, 4), p, d)
            blocks.route_experts(i(4, 2), f(4, 2), i(6), i(8), i(4, 2), f(4, 5))
            blocks.route_experts_gradient(f(4, 5), f(4, 2), f(4, 2), i(4, 2), f(4, 5), renormalize=False)
            blocks.grouped_gemm(f(8, 3), True, 1.0, f(4, 8), f(5, 3, 8), 0.0, i(6), index=i(8))
            blocks.grouped_gemm_weights(f(5, 3, 8), 1.0, f(8, 3), f(4, 8), 0.0, i(6), b_index=i(8))
            blocks.combine_experts(f(4, 8), f(8, 8), f(4, 2), i(4, 2))
            blocks.combine_experts_gradient(f(8, 8), f(4, 2), f(4, 8), f(8, 8), f(4, 2), i(4, 2))
        calls.append([(name, [a if isinstance(a, (int, float, str, tuple)) else None for a in args]) for name, args in stream.calls])
    assert calls[0] == calls[1] and len(calls[0]) == 8
    numbers = [a for _, args in calls[1][2:] for a in args if a is not None and not isinstance(a, (float, str))]
    assert all(type(a) in (int, bool) for a in numbers), numbers
