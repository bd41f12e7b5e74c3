"""Gradient optimizers of the tensor-math path: a Python mirror of
``src/cortex/optimize.clj:5-24``, ``src/cortex/optimize/adam.clj:116-200``,
``src/cortex/optimize/adadelta.clj:19-132`` and ``src/cortex/optimize/sgd.clj``.

An optimizer object implements ``PGradientOptimizer``: ``batch_update`` is
called once per batch, ``compute_parameters`` once per parameter buffer with
the running ``offset`` of that buffer inside the flat optimizer state
(``src/cortex/nn/compute_binding.clj:817-854``).  The Adam and Adadelta steps
are one fused kernel each on the backend's stream; SGD is, as in the reference,
four calls of the tensor API.  Muon, which the reference has not, is one call of
products between which nothing is done; it makes the momentum of a matrix
orthogonal (:func:`orthogonalize`).
"""
from __future__ import annotations

import array
import dataclasses

from . import capi
from . import dimensions as dims

# Of a step of :func:`orthogonalize`: odd polynomials of fifth degree whose slope at zero is large, so that small singular values
# grow soonest; what is above them ends between 0.7 and 1.2.
NEWTON_SCHULZ_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def adam(**kwargs) -> dict:
    """Default Adam description (``adam.clj:191-200``)."""
    out = {"type": "adam", "alpha": 0.001, "beta1": 0.9, "beta2": 0.999, "epsilon": 1e-8}
    out.update(kwargs)
    return out


def adadelta(**kwargs) -> dict:
    """Default Adadelta description (``adadelta.clj:124-132``)."""
    out = {"type": "adadelta", "decay": 0.05, "epsilon": 1e-6}
    out.update(kwargs)
    return out


def sgd(**kwargs) -> dict:
    """Default SGD description (``sgd.clj:74-80``)."""
    out = {"type": "sgd", "learning-rate": 0.001, "momentum": 0.9}
    out.update(kwargs)
    return out


def muon(**kwargs) -> dict:
    """Default Muon description: momentum whose matrices are made orthogonal before they are taken off the parameters (:class:`Muon`).
    No counterpart in the reference."""
    out = {"type": "muon", "alpha": 0.02, "momentum": 0.95, "nesterov": True, "steps": 5, "coefficients": NEWTON_SCHULZ_COEFFICIENTS,
           "epsilon": 1e-7, "weight-decay": 0.0}
    out.update(kwargs)
    return out


@dataclasses.dataclass
class Backend:
    """What the optimizers need of a compute backend: its stream and datatype
    (``src/cortex/compute/cuda/backend.clj:33-72``)."""
    stream: object
    datatype: str = "float"
    type: str = "hip"


def _buffer(x):
    return x.buffer if hasattr(x, "buffer") else x


def _dense_buffer(x):
    """(a buffer, the order of its elements) of a buffer, or of a tensor whose elements are all of it.  The order is None where
    they lie as they are counted; else (extent, stride) of every dimension but those of one element."""
    if not hasattr(x, "buffer"):
        return x, None
    shape, strides = x.dimensions["shape"], x.dimensions["strides"]
    n, dense, expected = x.ecount(), dims.direct_shape(shape), 1
    order = [(int(extent), int(stride)) for extent, stride in zip(shape, strides) if extent != 1] if n and dense else []
    for extent, stride in sorted(order, key=lambda d: d[1]):
        dense = dense and stride == expected
        expected *= extent
    if not dense:
        raise ValueError("clip_gradients: tensors must be dense")
    as_counted = all(a[1] > b[1] for a, b in zip(order, order[1:]))
    return x.buffer if x.buffer.ecount() == n else x.buffer.sub_buffer(0, n), None if as_counted else order


def _ensure_datatype(datatype, *buffers) -> None:
    actual = [b.get_datatype() for b in buffers]
    if any(a != datatype for a in actual):
        raise TypeError(f"Buffer datatype mismatch: expected {datatype}, got {actual}")


@dataclasses.dataclass
class Adam:
    backend: Backend
    optimizer: dict
    pow_beta1_t: float = 1.0
    pow_beta2_t: float = 1.0

    def batch_update(self, optimizer_parameters=None) -> "Adam":
        """``batch-update`` (``adam.clj:149-153``): beta^t by repeated multiplication."""
        return dataclasses.replace(self, pow_beta1_t=self.pow_beta1_t * float(self.optimizer["beta1"]),
                                   pow_beta2_t=self.pow_beta2_t * float(self.optimizer["beta2"]))

    def compute_parameters(self, state: dict, gradient_alpha, offset: int, gradient, parameters) -> None:
        """``compute-parameters!`` (``adam.clj:154-158`` -> ``adam-optimise-step!`` :116-134)."""
        g, p, m, v = _buffer(gradient), _buffer(parameters), _buffer(state["m"]), _buffer(state["v"])
        _ensure_datatype(self.backend.datatype, g, p, m, v)
        n = g.ecount()
        o = self.optimizer
        self.backend.stream.adam_step(o["alpha"], o["beta1"], o["beta2"], o["epsilon"], self.pow_beta1_t,
                                      self.pow_beta2_t, gradient_alpha, g, p,
                                      m.sub_buffer(offset, m.ecount() - offset),
                                      v.sub_buffer(offset, v.ecount() - offset), n)


@dataclasses.dataclass
class Adadelta:
    backend: Backend
    optimizer: dict

    def batch_update(self, optimizer_parameters=None) -> "Adadelta":
        return self

    def compute_parameters(self, state: dict, gradient_alpha, offset: int, gradient, parameters) -> None:
        """``compute-parameters!`` (``adadelta.clj:19-26``)."""
        g, p = _buffer(gradient), _buffer(parameters)
        ga, da = _buffer(state["grad-accum"]), _buffer(state["dx-accum"])
        _ensure_datatype(self.backend.datatype, g, p, ga, da)
        o = self.optimizer
        self.backend.stream.adadelta_step(o["decay"], o["epsilon"], ga.sub_buffer(offset, ga.ecount() - offset),
                                          da.sub_buffer(offset, da.ecount() - offset), gradient_alpha, g, p, g.ecount())


@dataclasses.dataclass
class SGD:
    backend: Backend
    optimizer: dict
    _temp: object = None   # the allocator's reusable :sgd-temp tensor (sgd.clj:27)

    def batch_update(self, optimizer_parameters=None) -> "SGD":
        return self

    def compute_parameters(self, state: dict, gradient_alpha, offset: int, gradient, parameters) -> None:
        """``tensor-sgd`` (``sgd.clj:16-40``): momentum with the look-ahead correction,
            dxm = momentum * v;  v = dxm + learning-rate * gradient-alpha * g;
            dx = dxm - (1 + momentum) * v;  p = p + dx
        as one ``unary-op!`` and three ``binary-op!`` calls."""
        from . import tensor as ct
        from . import dimensions as dims

        g, p, mv = _buffer(gradient), _buffer(parameters), _buffer(state["momentum-vals"])
        _ensure_datatype(self.backend.datatype, g, p, mv)
        n = g.ecount()
        device = self.backend.stream.get_device()
        vec = lambda buf, count: ct.Tensor(device, dims.dimensions([count]), buf)
        momentum = float(self.optimizer["momentum"])
        with ct.tensor_context(self.backend.stream, self.backend.datatype):
            grad, params = vec(g, n), vec(p, p.ecount())
            momentum_vals = vec(mv.sub_buffer(offset, n), n)
            if self._temp is None or self._temp.ecount() < n:
                self._temp = ct.new_tensor([n], init_value=None)
            temp = vec(self._temp.buffer.sub_buffer(0, n), n)
            dxm = ct.unary_op(temp, momentum, momentum_vals, "noop")
            ct.binary_op(momentum_vals, 1.0, dxm, float(self.optimizer["learning-rate"]) * float(gradient_alpha), grad, "+")
            dx = ct.binary_op(temp, 1.0, dxm, 1 + momentum, momentum_vals, "-")
            ct.binary_op(params, 1.0, params, 1.0, dx, "+")


def _matrices(name: str, what: str, x):
    """(matrices, rows, columns, distance of rows, distance of matrices) of a tensor of one matrix or of several."""
    if not hasattr(x, "buffer"):
        raise ValueError(f"{name}: {what} must be a tensor, whose shape says what its matrices are")
    shape, strides = x.dimensions["shape"], x.dimensions["strides"]
    if not 2 <= len(shape) <= 3 or not dims.direct_shape(shape):
        raise ValueError(f"{name}: {what} must be a matrix or matrices, got the shape {list(x.shape())}")
    shape, strides = [int(n) for n in shape], [int(n) for n in strides]
    if len(shape) == 2:
        shape, strides = [1, *shape], [0, *strides]
    count, rows, columns = shape
    if (columns > 1 and strides[2] != 1) or (rows > 1 and strides[1] < columns):
        raise ValueError(f"{name}: the rows of {what} must be contiguous and apart from one another")
    return count, rows, columns, max(strides[1], columns) if rows > 1 else columns, strides[0] if count > 1 else 0


def _packed_matrices(name: str, what: str, x, shape):
    found = _matrices(name, what, x)
    if found[:3] != shape or (0 not in shape and (found[3] != shape[2] or (shape[0] > 1 and found[4] != shape[1] * shape[2]))):
        raise ValueError(f"{name}: {what} must be dense and of shape {list(shape)}, got {list(x.shape())}")
    return x.buffer


def _steps_of(coefficients, steps: int) -> bytes:
    """Three doubles to a step: of one triple for all steps, or of one to each."""
    if not len(coefficients):
        raise ValueError("coefficients: none")
    triples = [tuple(map(float, c)) for c in coefficients] if hasattr(coefficients[0], "__len__") else [tuple(map(float, coefficients))] * int(steps)
    if len(triples) != int(steps) or any(len(c) != 3 for c in triples):
        raise ValueError(f"coefficients: three numbers, or three to each of {steps} steps")
    return array.array("d", [x for c in triples for x in c]).tobytes()


def orthogonalize_workspace(backend: Backend, input):
    """A buffer for :func:`orthogonalize` of such a tensor, as large as makes all of its launches fill the chip.  Calls that may
    overlap in time (on two streams, or of two recorded graphs) need one each; its owner releases it."""
    _ensure_datatype(backend.datatype, _buffer(input))
    need = backend.stream.orthogonalize_workspace(*_matrices("orthogonalize", "input", input)[:3], backend.datatype)
    return backend.stream.get_device().allocate_device_buffer(max(1, need), "byte")


def orthogonalize(backend: Backend, output, input, *, alpha=1.0, beta=0.0, steps: int = 5, coefficients=NEWTON_SCHULZ_COEFFICIENTS,
                  epsilon=1e-7, workspace=None) -> None:
    """output = alpha * (input made orthogonal) + beta * output, of a matrix or of each of several ([count, rows, columns]):

        X = input / (|input| + epsilon);   steps times, on the shorter side:  A = X X^T,  X = (a I + b A + c A A) X

    with |.| the root of the sum of squares and (a, b, c) the coefficients, one triple or one to a step.  Rows are contiguous and any
    distance apart; ``output`` may be ``input``.  ``workspace`` is of :func:`orthogonalize_workspace`; a smaller one serves as long as
    one matrix fits.  Without it one is allocated and released, which waits for the stream.  No counterpart in the reference."""
    name = "orthogonalize"
    of_input, of_output = _matrices(name, "input", input), _matrices(name, "output", output)
    if of_input[:3] != of_output[:3]:
        raise ValueError(f"{name}: output {list(output.shape())} and input {list(input.shape())} differ")
    _ensure_datatype(backend.datatype, output.buffer, input.buffer)
    if any(x.device is not output.buffer.device for x in (input.buffer, *([] if workspace is None else [_buffer(workspace)]))):
        raise ValueError(f"{name}: buffers are not all on the same device")
    steps_of = _steps_of(coefficients, steps)
    own = workspace is None
    if own:
        workspace = orthogonalize_workspace(backend, input)
    try:
        backend.stream.orthogonalize(output.buffer, *of_output[3:], alpha, input.buffer, *of_input[3:], beta, *of_input[:3], steps_of, epsilon,
                                     _buffer(workspace))
        if own:
            backend.stream.sync()
    finally:
        if own:
            workspace.release()


_MOST_GROWTH = 64 << 20


@dataclasses.dataclass
class Muon:
    """Momentum for matrices, made orthogonal before it is taken off the parameters: of a matrix [rows, columns]

        v = momentum * v + gradient-alpha * g;    u = gradient-alpha * g + momentum * v (nesterov), or v
        p = (1 - alpha * weight-decay) * p - alpha * sqrt(max(1, rows / columns)) * orthogonalize(u)

    in one call of the library.  Parameters are tensors [rows, columns], a row to an output, or [matrices, rows, columns], as those of
    experts are; vectors are for another optimizer.  What lies between the products is kept from step to step, and what was too small
    for a larger matrix is kept too: a recorded graph may still write to it.  A step that needs more than any before it allocates, so one is
    made before a graph of it is recorded; steps of one optimizer do not run on two streams at once."""
    backend: Backend
    optimizer: dict
    _workspaces: list = dataclasses.field(default_factory=list)
    _refused: int = None     # bytes that there was no memory for

    def batch_update(self, optimizer_parameters=None) -> "Muon":
        return self

    def _workspace(self, *shape):
        """A buffer for a step of such matrices, kept.  Small ones grow by twice at least, so that there are few; where there is no memory for as
        much as fills the chip, what one matrix takes serves, and the matrices take turns."""
        stream, have = self.backend.stream, self._workspaces[-1].ecount() if self._workspaces else 0
        need = max(1, stream.orthogonalize_workspace(*shape, self.backend.datatype))
        if have >= need:
            return self._workspaces[-1]
        least = max(1, stream.orthogonalize_workspace(min(shape[0], 1), *shape[1:], self.backend.datatype))
        sizes = [n for n in (max(need, min(2 * have, _MOST_GROWTH)), need) if n < (self._refused or n + 1)]
        for size in dict.fromkeys([*sizes, least]):
            if size <= have:
                break
            try:
                self._workspaces.append(stream.get_device().allocate_device_buffer(size, "byte"))
                break
            except capi.CortexHipError as e:
                if size == least or "out of memory" not in e.message:
                    raise
                self._refused = size     # asked for once: each further step would wait for the same answer
        return self._workspaces[-1]

    def compute_parameters(self, state: dict, gradient_alpha, offset: int, gradient, parameters) -> None:
        name, o, stream = "muon", self.optimizer, self.backend.stream
        shape = _matrices(name, "parameters", parameters)[:3]
        p = _packed_matrices(name, "parameters", parameters, shape)
        g = _packed_matrices(name, "gradient", gradient, shape) if hasattr(gradient, "buffer") else gradient
        v = _buffer(state["momentum-vals"])
        _ensure_datatype(self.backend.datatype, g, p, v)
        n = shape[0] * shape[1] * shape[2]
        if g.ecount() < n or p.ecount() < n:
            raise ValueError(f"{name}: parameters of shape {list(shape)} and a gradient of {g.ecount()} elements")
        if any(x.device is not p.device for x in (g, v)):
            raise ValueError(f"{name}: buffers are not all on the same device")
        steps_of = _steps_of(o["coefficients"], o["steps"])
        workspace = self._workspace(*shape)
        stream.muon_step(o["alpha"], o["momentum"], o["nesterov"], o["weight-decay"], gradient_alpha, steps_of, o["epsilon"], g, p,
                         v.sub_buffer(offset, n), *shape, workspace)


def clip_gradients(backend: Backend, gradients, max_norm, norm_and_factor, outputs=None, in_place: bool = True) -> None:
    """The norm over all ``gradients`` (buffers or dense tensors of the backend's datatype) and their clipping, ahead of
    ``compute_parameters``: with norm = sqrt(sum of all squares),

        factor = max_norm / max(norm, max_norm),   outputs = gradients * factor

    into ``outputs`` (each in the order of its gradient, where that is not the order of its elements) or, without them, into the gradients themselves; with ``in_place`` false and no outputs only the norm
    is formed.  ``norm_and_factor`` holds two values on the device, so that nothing waits for the host.  The reference's
    gradients are sums over a batch that an optimizer multiplies by its gradient-alpha: a limit for their mean is the
    batch's size times as much.  No counterpart in the reference."""
    result, _ = _dense_buffer(norm_and_factor)
    if result.ecount() != 2:
        raise ValueError("clip_gradients: the norm and the factor are two values")
    if not float(max_norm) > 0:
        raise ValueError(f"clip_gradients: max_norm must be positive, got {max_norm}")
    at, counts, datatype, orders = _addresses(gradients, backend.datatype)
    into = at if in_place else None
    if outputs is not None:
        into, of_outputs, other, into_orders = _addresses(outputs, backend.datatype)
        if of_outputs != counts:
            raise ValueError("clip_gradients: outputs and gradients differ in their lengths")
        if into_orders != orders:
            raise ValueError("clip_gradients: the elements of an output lie in another order than its gradient's")
        if other != datatype:
            raise TypeError(f"Buffer datatype mismatch: expected {backend.datatype}, got {[datatype, other]}")
    _ensure_datatype(backend.datatype, result)
    if datatype != backend.datatype:
        raise TypeError(f"Buffer datatype mismatch: expected {backend.datatype}, got {datatype}")
    backend.stream.clip_gradients(at, counts, into, max_norm, result)


def _addresses(tensors, datatype):
    """(device addresses, lengths, datatype, orders) of buffers or dense tensors: bytes of eight to each of the first two; the
    orders are None where all lie as they are counted, which is what native code takes."""
    if capi.front is not None:
        found = capi.front.addresses(tensors)    # 0.2 us to a tensor, 1 us here
        if found is not None:
            return (*found, None)
    found = [_dense_buffer(x) for x in tensors]
    buffers, orders = [b for b, _ in found], [order for _, order in found]
    _ensure_datatype(datatype, *buffers)
    return (array.array("Q", [b.ptr for b in buffers]).tobytes(), array.array("q", [b.ecount() for b in buffers]).tobytes(), datatype,
            orders if any(order is not None for order in orders) else None)


def create_optimizer(backend: Backend, optimizer: dict):
    """``create-optimizer`` multimethod on ``[(:type backend) (:type optimizer)]``
    (``optimize.clj:19-24``)."""
    if backend.datatype not in ("float", "double"):
        raise TypeError("optimizers support float and double only")
    kind = optimizer["type"]
    if kind == "adam":
        return Adam(backend, optimizer)
    if kind == "adadelta":
        return Adadelta(backend, optimizer)
    if kind == "sgd":
        return SGD(backend, optimizer)
    if kind == "muon":
        return Muon(backend, optimizer)
    raise KeyError(f"No optimizer {kind!r} for backend {backend.type!r}")
