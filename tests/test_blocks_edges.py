"""Calls of the operators of residual blocks with experts that are refused, or that reach the stream, by how their operands lie
in memory.  Nothing here needs a GPU."""
import struct

import pytest

from cortex_amd import capi
from cortex_amd import optimize
from cortex_amd import tensor as ct
from test_blocks_refusals import Recorder, t


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
def test_clipping_takes_tensors_that_fill_their_memory(native, monkeypatch):
    """A row that is given again and again, or rows apart: what lies between is no gradient."""
    if not native:
        monkeypatch.setattr(capi, "front", None)
    for shape, strides in (([4, 4], [4, 0]), ([4, 4], [8, 1]), ([2, 3], [3, 2])):
        with pytest.raises(ValueError, match="must be dense"):
            clipped([at(4096, *shape, strides=strides, count=100)])
