"""The memory that an optimizer for matrices keeps: what is asked of the device, step by step.  Nothing here needs a GPU."""
import pytest

from cortex_amd import capi
from cortex_amd import optimize
from test_orthogonalize_refusals import Buffer, matrix


class Device:
    """Memory of `room` bytes; what is asked of it is recorded."""

    def __init__(self, room, message="hipMalloc failed: out of memory"):
        self.room, self.asked, self.message = room, [], message

    def allocate_device_buffer(self, n, datatype):
        assert datatype == "byte"
        self.asked.append(n)
        if n > self.room:
            raise capi.CortexHipError(2, self.message)
        self.room -= n
        return Buffer(n, datatype)


class Stream:
    """A step needs a MiB to each 1024 elements of a matrix."""

    def __init__(self, device):
        self.device, self.given = device, []

    def get_device(self):
        return self.device

    def orthogonalize_workspace(self, count, rows, columns, datatype):
        return count * rows * columns << 10

    def muon_step(self, *args):
        self.given.append(args[-1].ecount())


def steps(room, *shapes, message=None):
    device = Device(room, *([message] if message else []))
    stream = Stream(device)
    optimizer = optimize.create_optimizer(optimize.Backend(stream, "float"), optimize.muon())
    for shape in shapes:
        n = shape[0] * shape[1] * shape[2]
        optimizer.compute_parameters({"momentum-vals": Buffer(n)}, 1.0, 0, matrix(*shape), matrix(*shape))
    return device.asked, stream.given


MIB = 1 << 20


def test_small_ones_double_and_large_ones_are_as_large_as_they_need_to_be():
    asked, given = steps(1 << 40, (1, 32, 32), (1, 32, 33), (1, 64, 32), (4, 1024, 1024), (4, 1024, 1025), (1, 32, 32))
    assert asked == [MIB, 2 * MIB, 4 * 1024 * MIB, 4 * 1025 * MIB]      # 64 x 32 fits what the second one doubled to
    assert given == [MIB, 2 * MIB, 2 * MIB, 4 * 1024 * MIB, 4 * 1025 * MIB, 4 * 1025 * MIB]


def test_where_there_is_no_memory_the_matrices_take_turns():
    asked, given = steps(10 * MIB, (8, 32, 64), (8, 32, 64), (1, 32, 64))
    assert given == [2 * MIB] * 3
    assert asked == [16 * MIB, 2 * MIB]      # asked once, not at every step
    # what fits is taken, without what it would have doubled to
    asked, given = steps(12 * MIB, (4, 32, 32), (5, 32, 32))
    assert asked == [4 * MIB, 8 * MIB] and given == [4 * MIB, 8 * MIB]
    asked, given = steps(11 * MIB, (4, 32, 32), (5, 32, 32))
    assert asked == [4 * MIB, 8 * MIB, 5 * MIB] and given == [4 * MIB, 5 * MIB]
    # what is there serves, if it is no less than one matrix takes
    asked, given = steps(5 * MIB, (4, 32, 32), (6, 32, 32), (6, 32, 32))
    assert asked == [4 * MIB, 8 * MIB, 6 * MIB] and given == [4 * MIB] * 3


def test_where_not_even_one_matrix_fits():
    with pytest.raises(capi.CortexHipError, match="out of memory"):
        steps(MIB, (8, 32, 64))
    with pytest.raises(capi.CortexHipError, match="capturing"):      # any other refusal is not tried again with less
        steps(0, (8, 32, 64), message="operation not permitted when stream is capturing")
