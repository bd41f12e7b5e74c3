"""Residual feed-forward blocks, dense and with experts: the operators that such a block with norms around it is trained and
served with, in the manner of the tensor API (:mod:`cortex_amd.tensor`), and layers that run them together
(:class:`GatedBlock`, :class:`ExpertBlock`).  No counterpart in the reference.

    output, normalized = norm_residual(block's result, residual)    the norms after a block and before the next one
    gated_gemm                                                      both first projections of rows, and f(gate) * up
    route_experts(normalized x router)                              the experts of each token, and rows in their order
    grouped_gemm                                                    products of rows with their expert's matrix
    combine_experts                                                 the weighted sum of a token's rows

Every call has its gradient next to it.  Tensors are float or double; those of indexes are int.  Matrices are row-major with
unit stride along a row; rows may lie any distance apart (``submatrix``).  Clipping by the norm of all gradients is with the
optimizers (:func:`cortex_amd.optimize.clip_gradients`).
"""
from __future__ import annotations

from . import capi
from . import dimensions as dims
from . import tensor as ct
from .tensor import Tensor, TensorError, check_stream

# What the operands of a call are, found in native code (csrc/front.cpp) where they are as they mostly are: each call checks
# those numbers, and what does not pass there goes through the checks below, which say what is wrong.  (Some 10 us of Python a
# call, for kernels of 3 to 5; 2 us so.)
_operands = capi.front.operands if capi.front is not None else lambda kinds, tensors: None

NORM_KINDS = ("none", "rms", "layer")


def _floating(name: str, first: Tensor, *others) -> None:
    datatype = first.get_datatype()
    if datatype not in ("float", "double"):
        raise TensorError(f"{name} is only defined for float and double tensors")
    for t in others:
        if t is None:
            continue
        if t.get_datatype() != datatype:
            raise TensorError(f"{name}: not all arguments match required datatype {datatype}")
        if t.device is not first.device:
            raise TensorError("Tensor arguments are not all on same device")


def _needed(name: str, **tensors) -> None:
    for what, t in tensors.items():
        if t is None:
            raise TensorError(f"{name}: {what.replace('_', ' ')} is needed")


def _is_packed(t: Tensor) -> bool:
    shape, expected = t.dimensions["shape"], 1
    if not dims.direct_shape(shape):
        return False
    if 0 in shape:    # whatever its strides
        return True
    for n, stride in zip(reversed(shape), reversed(t.dimensions["strides"])):
        if n != 1 and stride != expected:
            return False
        expected *= n
    return True


def _indexes(name: str, first: Tensor, **tensors) -> None:
    for what, t in tensors.items():
        if t is None:
            continue
        if t.get_datatype() != "int":
            raise TensorError(f"{name}: {what} must be an int tensor")
        if not _is_packed(t):
            raise TensorError(f"{name}: {what} must be dense")
        if t.device is not first.device:
            raise TensorError("Tensor arguments are not all on same device")


def _packed(name: str, what: str, t: Tensor, shape) -> Tensor:
    if t is not None and (list(t.shape()) != list(shape) or not _is_packed(t)):
        raise TensorError(f"{name}: {what} must be a dense tensor of shape {list(shape)}, got {list(t.shape())}")
    return t


def _rows(name: str, what: str, t: Tensor):
    """(rows, columns, distance of rows) of a matrix whose rows are contiguous; a vector is one row."""
    shape, strides = t.dimensions["shape"], t.dimensions["strides"]
    if not 1 <= len(shape) <= 2 or not dims.direct_shape(shape):
        raise TensorError(f"{name}: {what} must be a matrix")
    shape, strides = [int(n) for n in shape], [int(n) for n in strides]
    if len(shape) == 1:
        shape, strides = [1, shape[0]], [shape[0], strides[0]]
    rows, columns = shape
    if columns > 1 and strides[1] != 1:
        raise TensorError(f"{name}: the rows of {what} must be contiguous")
    stride = strides[0] if rows > 1 else max(strides[0], columns)
    if stride < columns:
        raise TensorError(f"{name}: the rows of {what} overlap")
    return rows, columns, stride


def _buffer(t: Tensor):
    return None if t is None else t.buffer


def _dims(t: Tensor):
    return None if t is None else t.dimensions


# ---------------------------------------------------------------- norms, gate and residual

def norm_descriptor(*, post="rms", pre="rms", epsilon=1e-5, residual_scale=1.0) -> dict:
    """The norms after a block (``post``) and before the next one (``pre``), each "rms", "layer" or "none", and what the
    residual is multiplied by.  The library keeps no native object for it."""
    for kind in (post, pre):
        if kind not in NORM_KINDS:
            raise TensorError(f"Unrecognized norm {kind!r}: one of {NORM_KINDS}")
    if not float(epsilon) >= 0:
        raise TensorError("Epsilon must not be negative")
    return {"post": post, "pre": pre, "epsilon": float(epsilon), "residual-scale": float(residual_scale)}


_OF_COLUMNS = ("post-scale", "post-bias", "pre-scale", "pre-bias")
_PARAMETERS = {*_OF_COLUMNS, "gate"}


def _norm_fits(shape, matrices, gate, statistics, scales) -> bool:
    """Whether matrices (rows, columns, distance; zeros if absent) are of ``shape`` and the other operands go with it."""
    rows, columns = shape
    for i in range(0, len(matrices), 3):
        if matrices[i] and (matrices[i] != rows or matrices[i + 1] != columns):
            return False
    if gate[0] and not (gate[0] in (1, rows) and gate[1] in (1, columns)):
        return False
    if statistics[0] and statistics != (2, 4 * rows, rows):
        return False
    for i in range(0, len(scales), 3):
        if scales[i] and (scales[i] != 1 or scales[i + 1] != columns):
            return False
    return True


def _norm_parameters(name: str, first: Tensor, parameters: dict, shape):
    unknown = set(parameters) - set(_OF_COLUMNS) - {"gate"}
    if unknown:
        raise TensorError(f"{name}: unknown parameters {sorted(unknown)}")
    _floating(name, first, *parameters.values())
    for key in _OF_COLUMNS:
        _packed(name, key, parameters.get(key), [shape[1]])
    gate = parameters.get("gate")
    if gate is not None:
        rows, columns, _ = _rows(name, "gate", gate)
        if rows not in (1, shape[0]) or columns not in (1, shape[1]):
            raise TensorError(f"{name}: the gate's shape {list(gate.shape())} does not go with {list(shape)}")
    return gate


def norm_residual(output: Tensor, normalized: Tensor, statistics: Tensor, input: Tensor, residual: Tensor, parameters: dict,
                  descriptor: dict):
    """What leaves a block and enters the next one, in one pass:

        output = residual-scale * residual + gate * (N_post(input) * post-scale + post-bias)
        normalized = N_pre(output) * pre-scale + pre-bias

    ``parameters`` may hold "post-scale", "post-bias", "pre-scale", "pre-bias" ([width]) and "gate" ([rows, width], or 1 in
    either place); ``residual`` may be None, ``normalized`` too without a norm before the next block.  ``statistics``
    ([4, rows], or None) is what :func:`norm_residual_gradient` needs.  ``output`` and ``normalized`` may each be the residual or
    the input itself."""
    name = "norm-residual"
    p = parameters.get
    has_pre = descriptor["pre"] != "none"
    if output is not None and parameters.keys() <= _PARAMETERS and (normalized is not None or not has_pre):
        normalized = normalized if has_pre else None
        gate, scales = p("gate"), (p("post-scale"), p("post-bias"), p("pre-scale"), p("pre-bias"))
        found = _operands("mmmmmppppp", (input, output, residual, normalized, gate, statistics, *scales))
        if found is not None and _norm_fits(found[:2], found[3:12], found[12:15], found[15:18], found[18:]):
            check_stream().norm_residual(output.buffer, output.dimensions, _buffer(normalized), _dims(normalized), _buffer(statistics),
                                         input.buffer, input.dimensions, _buffer(residual), _dims(residual), _buffer(gate),
                                         _dims(gate), *map(_buffer, scales), descriptor["post"], descriptor["pre"],
                                         descriptor["residual-scale"], descriptor["epsilon"])
            return output, normalized
    _needed(name, input=input, output=output)
    shape = _rows(name, "input", input)[:2]
    if has_pre and normalized is None:
        raise TensorError(f"{name}: a norm before the next block needs a tensor to store to")
    normalized = normalized if has_pre else None
    _floating(name, output, normalized, statistics, input, residual)
    for what, t in (("output", output), ("normalized", normalized), ("residual", residual)):
        if t is not None and _rows(name, what, t)[:2] != shape:
            raise TensorError(f"{name}: shapes differ: {what} {list(t.shape())}, input {list(shape)}")
    _packed(name, "statistics", statistics, [4, shape[0]])
    gate = _norm_parameters(name, output, parameters, shape)
    check_stream().norm_residual(output.buffer, output.dimensions, _buffer(normalized), _dims(normalized), _buffer(statistics),
                                 input.buffer, input.dimensions, _buffer(residual), _dims(residual), _buffer(gate), _dims(gate),
                                 _buffer(p("post-scale")), _buffer(p("post-bias")), _buffer(p("pre-scale")),
                                 _buffer(p("pre-bias")), descriptor["post"], descriptor["pre"], descriptor["residual-scale"],
                                 descriptor["epsilon"])
    return output, normalized


def norm_residual_gradient(input_gradient: Tensor, residual_gradient: Tensor, parameter_gradients: dict, output_gradient: Tensor,
                           normalized_gradient: Tensor, input: Tensor, output: Tensor, statistics: Tensor, parameters: dict,
                           descriptor: dict):
    """The gradients of :func:`norm_residual`, all overwritten, from those of its results (either may be None: zero).  Any
    gradient that is None, or not in ``parameter_gradients``, is not formed."""
    name = "norm-residual-gradient"
    p, g = parameters.get, parameter_gradients.get
    if parameters.keys() <= _PARAMETERS and parameter_gradients.keys() <= parameters.keys():
        gate, scales = p("gate"), (p("post-scale"), p("post-bias"), p("pre-scale"), p("pre-bias"))
        results = (g("post-scale"), g("post-bias"), g("pre-scale"), g("pre-bias"))
        found = _operands("mmmmmmmmppppppppp", (input, input_gradient, residual_gradient, output_gradient, normalized_gradient,
                                                output, gate, g("gate"), statistics, *scales, *results))
        if (found is not None and _norm_fits(found[:2], found[3:18], found[18:21], found[24:27], found[27:]) and
                (not found[21] or (found[21:23] == found[18:20] and found[23] == found[22])) and
                not any(b and not a for a, b in zip(found[27:39:3], found[39::3]))):
            check_stream().norm_residual_gradient(
                _buffer(input_gradient), _dims(input_gradient), _buffer(residual_gradient), _dims(residual_gradient),
                _buffer(g("gate")), *map(_buffer, results), _buffer(output_gradient), _dims(output_gradient),
                _buffer(normalized_gradient), _dims(normalized_gradient), input.buffer, input.dimensions, _buffer(output),
                _dims(output), _buffer(statistics), _buffer(gate), _dims(gate), *map(_buffer, scales[:3]), descriptor["post"],
                descriptor["pre"], descriptor["residual-scale"])
            return input_gradient, residual_gradient
    _needed(name, input=input)
    shape = _rows(name, "input", input)[:2]
    _floating(name, input, input_gradient, residual_gradient, output_gradient, normalized_gradient, output, statistics)
    for what, t in (("input gradient", input_gradient), ("residual gradient", residual_gradient),
                    ("output gradient", output_gradient), ("normalized gradient", normalized_gradient), ("output", output)):
        if t is not None and _rows(name, what, t)[:2] != shape:
            raise TensorError(f"{name}: shapes differ: {what} {list(t.shape())}, input {list(shape)}")
    _packed(name, "statistics", statistics, [4, shape[0]])
    gate = _norm_parameters(name, input, parameters, shape)
    _floating(name, input, *parameter_gradients.values())
    for key, t in parameter_gradients.items():
        if t is None:
            continue
        if parameters.get(key) is None:
            raise TensorError(f"{name}: a gradient of {key!r}, which is no parameter")
        _packed(name, f"the gradient of {key}", t, parameters[key].shape())
    check_stream().norm_residual_gradient(
        _buffer(input_gradient), _dims(input_gradient), _buffer(residual_gradient), _dims(residual_gradient), _buffer(g("gate")),
        _buffer(g("post-scale")), _buffer(g("post-bias")), _buffer(g("pre-scale")), _buffer(g("pre-bias")),
        _buffer(output_gradient), _dims(output_gradient), _buffer(normalized_gradient), _dims(normalized_gradient), input.buffer,
        input.dimensions, _buffer(output), _dims(output), _buffer(statistics), _buffer(gate), _dims(gate),
        _buffer(p("post-scale")), _buffer(p("post-bias")), _buffer(p("pre-scale")), descriptor["post"], descriptor["pre"],
        descriptor["residual-scale"])
    return input_gradient, residual_gradient


# ---------------------------------------------------------------- the choice of experts

def route_experts(experts: Tensor, weights: Tensor, offsets: Tensor, tokens: Tensor, slots: Tensor, logits: Tensor, *,
                  renormalize: bool = True):
    """The experts of every token and the order of rows by expert, from ``logits`` [n, experts].

    ``experts`` and ``weights`` [n, chosen]: the largest logits, largest first, the lowest index first among equal ones, and
    their softmax, over themselves (``renormalize``) or over all logits.  A logit of -infinity is never chosen; where too
    few are left the expert is -1 and its weight 0.
    ``offsets`` [experts + 1], ``tokens`` [n * chosen], ``slots`` [n, chosen]: the assignments in order of their expert;
    expert e has the places offsets[e] to offsets[e + 1] - 1, ``tokens`` names the token at a place (-1 beyond the last
    one) and ``slots`` the place of an assignment (-1 where there is none)."""
    name = "route-experts"
    found = _operands("mipiii", (logits, experts, weights, offsets, tokens, slots))
    if found is not None:
        n, n_experts, stride, dimensions, count, n_chosen = found[:6]
        of_choice = (dimensions, count, n_chosen)
        if (dimensions == 2 and count == n * n_chosen and n_chosen <= 32 and n_chosen <= n_experts <= 1024 and
                found[6:9] == of_choice and found[9:12] == (1, n_experts + 1, n_experts + 1) and found[12:15] == (1, count, count) and
                found[15:] == of_choice):
            check_stream().route_experts(experts.buffer, weights.buffer, offsets.buffer, tokens.buffer, slots.buffer, logits.buffer,
                                         stride, n, n_experts, n_chosen, renormalize)
            return experts, weights
    _needed(name, logits=logits, experts=experts, weights=weights, offsets=offsets, tokens=tokens, slots=slots)
    n, n_experts, stride = _rows(name, "logits", logits)
    n_chosen = int(experts.shape()[-1])
    _floating(name, logits, weights)
    _indexes(name, logits, experts=experts, offsets=offsets, tokens=tokens, slots=slots)
    if not 1 <= n_chosen <= min(32, n_experts) or n_experts > 1024:
        raise TensorError(f"{name}: {n_chosen} of {n_experts} experts: 1 to 32 of at most 1024 are taken")
    for what, t, shape in (("experts", experts, [n, n_chosen]), ("weights", weights, [n, n_chosen]), ("slots", slots, [n, n_chosen]),
                           ("offsets", offsets, [n_experts + 1]), ("tokens", tokens, [n * n_chosen])):
        _packed(name, what, t, shape)
    check_stream().route_experts(experts.buffer, weights.buffer, offsets.buffer, tokens.buffer, slots.buffer, logits.buffer, stride,
                                 n, n_experts, n_chosen, renormalize)
    return experts, weights


def route_experts_gradient(logits_gradient: Tensor, weights_gradient: Tensor, weights: Tensor, experts: Tensor, logits: Tensor, *,
                           renormalize: bool = True) -> Tensor:
    """The gradient of the weights with respect to the logits, overwritten.  ``logits`` may be None under ``renormalize``."""
    name = "route-experts-gradient"
    found = _operands("mmppi", (logits_gradient, logits, weights_gradient, weights, experts))
    if found is not None:
        n, n_experts, gradient_stride, rows, columns, stride = found[:6]
        of_choice = found[12:]
        if ((found[3:5] == found[:2] or (logits is None and renormalize)) and of_choice[0] == 2 and of_choice[1] == n * of_choice[2] and
                found[6:9] == of_choice == found[9:12]):
            check_stream().route_experts_gradient(logits_gradient.buffer, gradient_stride, weights_gradient.buffer, weights.buffer,
                                                  experts.buffer, _buffer(logits), stride, n, n_experts, of_choice[2], renormalize)
            return logits_gradient
    _needed(name, logits_gradient=logits_gradient, weights_gradient=weights_gradient, weights=weights, experts=experts)
    n, n_experts, gradient_stride = _rows(name, "logits gradient", logits_gradient)
    n_chosen = int(experts.shape()[-1])
    _floating(name, logits_gradient, weights_gradient, weights, logits)
    _indexes(name, logits_gradient, experts=experts)
    for what, t in (("experts", experts), ("weights", weights), ("weights gradient", weights_gradient)):
        _packed(name, what, t, [n, n_chosen])
    stride = 0
    if logits is not None:
        if _rows(name, "logits", logits)[:2] != (n, n_experts):
            raise TensorError(f"{name}: logits {list(logits.shape())} and their gradient {list(logits_gradient.shape())} differ")
        stride = _rows(name, "logits", logits)[2]
    elif not renormalize:
        raise TensorError(f"{name}: the logits are needed")
    check_stream().route_experts_gradient(logits_gradient.buffer, gradient_stride, weights_gradient.buffer, weights.buffer,
                                          experts.buffer, _buffer(logits), stride, n, n_experts, n_chosen, renormalize)
    return logits_gradient


# ---------------------------------------------------------------- products by expert

def _matrices(name: str, what: str, t: Tensor):
    """(groups, rows, columns, distance of rows, distance of matrices) of a tensor of one matrix to a group."""
    shape, strides = t.dimensions["shape"], t.dimensions["strides"]
    if len(shape) != 3 or not dims.direct_shape(shape):
        raise TensorError(f"{name}: {what} must hold a matrix to each group")
    shape, strides = [int(n) for n in shape], [int(n) for n in strides]
    if (shape[2] > 1 and strides[2] != 1) or (shape[1] > 1 and strides[1] < shape[2]):
        raise TensorError(f"{name}: the rows of {what} must be contiguous")
    return (*shape, max(strides[1], shape[2]), strides[0])


def grouped_gemm(C: Tensor, trans_b, alpha, A: Tensor, B: Tensor, beta, offsets: Tensor, index: Tensor = None) -> Tensor:
    """For every group e and every row i in offsets[e] .. offsets[e + 1] - 1:
    C[i] = alpha * A[index[i]] * (trans-b? B[e]) + beta * C[i].  Rows of no group are left as they are.  Without ``index``
    row i of A is row i; an index outside A is a row of zeros."""
    name = "grouped-gemm"
    found = _operands("mmgii", (C, A, B, offsets, index))
    if found is not None:
        rows, columns, c_stride, a_rows, a_columns, a_stride, groups, b_rows, b_columns, b_row_stride, b_stride = found[:11]
        if ((b_rows, b_columns) == ((columns, a_columns) if trans_b else (a_columns, columns)) and
                found[11:14] == (1, groups + 1, groups + 1) and (found[14:] == (1, rows, rows) if index is not None else a_rows == rows)):
            check_stream().grouped_gemm(C.buffer, c_stride, trans_b, alpha, A.buffer, a_rows, a_columns, a_stride, _buffer(index),
                                        B.buffer, columns, b_row_stride, b_stride, offsets.buffer, groups, rows, beta)
            return C
    _needed(name, C=C, A=A, B=B, offsets=offsets)
    _floating(name, C, A, B)
    rows, c_columns, c_stride = _rows(name, "C", C)
    a_rows, a_columns, a_stride = _rows(name, "A", A)
    groups, b_rows, b_columns, b_row_stride, b_stride = _matrices(name, "B", B)
    _indexes(name, C, offsets=offsets, index=index)
    if trans_b:
        b_rows, b_columns = b_columns, b_rows
    if a_columns != b_rows or b_columns != c_columns:
        raise TensorError(f"{name}: {a_columns} columns of A, {b_rows} by {b_columns} of B and {c_columns} of C do not go together")
    _packed(name, "offsets", offsets, [groups + 1])
    if index is not None:
        _packed(name, "index", index, [rows])
    elif a_rows != rows:
        raise TensorError(f"{name}: A has {a_rows} rows, C {rows}")
    check_stream().grouped_gemm(C.buffer, c_stride, trans_b, alpha, A.buffer, a_rows, a_columns, a_stride, _buffer(index), B.buffer,
                                b_columns, b_row_stride, b_stride, offsets.buffer, groups, rows, beta)
    return C


def grouped_gemm_weights(C: Tensor, alpha, A: Tensor, B: Tensor, beta, offsets: Tensor, a_index: Tensor = None,
                         b_index: Tensor = None) -> Tensor:
    """For every group e: C[e] = alpha * sum over its rows i of A[a-index[i]]^T B[b-index[i]] + beta * C[e]; beta * C[e]
    where it has none."""
    name = "grouped-gemm-weights"
    found = _operands("mmgiii", (A, B, C, offsets, a_index, b_index))
    if found is not None:
        a_rows, a_columns, a_stride, b_rows, b_columns, b_stride, groups, c_rows, c_columns, c_row_stride, c_stride = found[:11]
        rows = found[15] if a_index is not None else a_rows
        if ((a_columns, b_columns) == (c_rows, c_columns) and found[11:14] == (1, groups + 1, groups + 1) and
                rows == (found[18] if b_index is not None else b_rows)):
            check_stream().grouped_gemm_weights(C.buffer, c_row_stride, c_stride, alpha, A.buffer, a_rows, a_columns, a_stride,
                                                _buffer(a_index), B.buffer, b_rows, b_columns, b_stride, _buffer(b_index),
                                                offsets.buffer, groups, rows, beta)
            return C
    _needed(name, C=C, A=A, B=B, offsets=offsets)
    _floating(name, C, A, B)
    groups, c_rows, c_columns, c_row_stride, c_stride = _matrices(name, "C", C)
    a_rows, a_columns, a_stride = _rows(name, "A", A)
    b_rows, b_columns, b_stride = _rows(name, "B", B)
    _indexes(name, C, offsets=offsets, a_index=a_index, b_index=b_index)
    if (a_columns, b_columns) != (c_rows, c_columns):
        raise TensorError(f"{name}: {a_columns} columns of A and {b_columns} of B do not go with {c_rows} by {c_columns} of C")
    _packed(name, "offsets", offsets, [groups + 1])
    counts = {(t.ecount() if t is not None else n) for t, n in ((a_index, a_rows), (b_index, b_rows))}
    if len(counts) != 1:
        raise TensorError(f"{name}: A and B have different numbers of rows: {sorted(counts)}")
    check_stream().grouped_gemm_weights(C.buffer, c_row_stride, c_stride, alpha, A.buffer, a_rows, a_columns, a_stride,
                                        _buffer(a_index), B.buffer, b_rows, b_columns, b_stride, _buffer(b_index), offsets.buffer,
                                        groups, counts.pop(), beta)
    return C


# ---------------------------------------------------------------- gated products

GATES = tuple(capi.GATE_OPS)


def _gate(name: str, activation) -> None:
    if activation not in capi.GATE_OPS:
        raise TensorError(f"{name}: unrecognized activation {activation!r}: one of {GATES}")


def _weights(name: str, what: str, t: Tensor, offsets):
    """As _matrices, of one matrix where there are no groups."""
    if offsets is not None:
        return _matrices(name, what, t)
    if len(t.dimensions["shape"]) != 2:
        raise TensorError(f"{name}: {what} must be a matrix where there are no offsets")
    return (1, *_rows(name, what, t), 0)


def gated_gemm(inner: Tensor, pre: Tensor, A: Tensor, B: Tensor, offsets: Tensor = None, index: Tensor = None, *,
               activation: str = "swish") -> Tensor:
    """inner[i] = f(gate) * up with [gate up] = A[index[i]] * transpose(B), B [2 * hidden, width] the gate's projection above the
    other's; with ``offsets`` B is [groups, 2 * hidden, width] and a row's is that of its group, as in :func:`grouped_gemm`.  ``pre``
    [rows, 2 * hidden] takes [gate up], which :func:`gated_gemm_gradient` needs; None where there is no backward pass.  ``activation`` is
    one of "logistic", "tanh", "relu", "swish" and "gelu"."""
    name = "gated-gemm"
    _gate(name, activation)
    grouped = offsets is not None
    found = _operands("mmmgii" if grouped else "mmmmii", (inner, pre, A, B, offsets, index))
    if found is not None:
        rows, hidden, stride, pre_rows, pre_columns, pre_stride, a_rows, a_columns, a_stride = found[:9]
        groups, b_rows, b_columns, b_row_stride, b_stride = found[9:14] if grouped else (1, *found[9:12], 0)
        of_offsets, of_index = found[14:17] if grouped else None, found[-3:]
        if ((b_rows, b_columns) == (2 * hidden, a_columns) and (pre is None or (pre_rows, pre_columns) == (rows, 2 * hidden)) and
                (not grouped or of_offsets == (1, groups + 1, groups + 1)) and (of_index == (1, rows, rows) if index is not None else a_rows == rows)):
            check_stream().gated_gemm(inner.buffer, stride, _buffer(pre), pre_stride, activation, A.buffer, a_rows, a_columns, a_stride,
                                      _buffer(index), B.buffer, hidden, b_row_stride, b_stride, _buffer(offsets), groups, rows)
            return inner
    _needed(name, inner=inner, A=A, B=B)
    _floating(name, inner, pre, A, B)
    _indexes(name, inner, offsets=offsets, index=index)
    rows, hidden, stride = _rows(name, "inner", inner)
    a_rows, a_columns, a_stride = _rows(name, "A", A)
    groups, b_rows, b_columns, b_row_stride, b_stride = _weights(name, "B", B, offsets)
    if (b_rows, b_columns) != (2 * hidden, a_columns):
        raise TensorError(f"{name}: {a_columns} columns of A, {b_rows} by {b_columns} of B and {hidden} of inner do not go together")
    pre_stride = 0
    if pre is not None:
        pre_rows, pre_columns, pre_stride = _rows(name, "pre", pre)
        if (pre_rows, pre_columns) != (rows, 2 * hidden):
            raise TensorError(f"{name}: pre must be {rows} by {2 * hidden}, got {list(pre.shape())}")
    if offsets is not None:
        _packed(name, "offsets", offsets, [groups + 1])
    if index is not None:
        _packed(name, "index", index, [rows])
    elif a_rows != rows:
        raise TensorError(f"{name}: A has {a_rows} rows, inner {rows}")
    check_stream().gated_gemm(inner.buffer, stride, _buffer(pre), pre_stride, activation, A.buffer, a_rows, a_columns, a_stride, _buffer(index),
                              B.buffer, hidden, b_row_stride, b_stride, _buffer(offsets), groups, rows)
    return inner


def gated_gemm_gradient(pre_gradient: Tensor, inner: Tensor, output_gradient: Tensor, B: Tensor, pre: Tensor, offsets: Tensor = None, *,
                        activation: str = "swish") -> Tensor:
    """What the backward pass of a gated block begins with.  From the gradient of the rows inner[i] * transpose(B), B [width, hidden] the
    projection back (or [groups, width, hidden]), with d = output-gradient[i] * B:

        pre-gradient[i] = [d * up * f'(gate)   d * f(gate)],    [gate up] = pre[i]

    and, unless it is None, inner[i] = f(gate) * up once more.  ``pre_gradient`` may be ``pre`` itself.  The gradients of the first
    products' operands are products of ``pre_gradient`` (gemm, or grouped_gemm and grouped_gemm_weights)."""
    name = "gated-gemm-gradient"
    _gate(name, activation)
    grouped = offsets is not None
    found = _operands("mmmmgi" if grouped else "mmmmmi", (pre_gradient, inner, output_gradient, pre, B, offsets))
    if found is not None:
        rows, columns, stride, inner_rows, inner_columns, inner_stride, a_rows, width, a_stride, pre_rows, pre_columns, pre_stride = found[:12]
        groups, b_rows, hidden, b_row_stride, b_stride = found[12:17] if grouped else (1, *found[12:15], 0)
        if ((rows, columns) == (pre_rows, pre_columns) == (a_rows, 2 * hidden) and b_rows == width and
                (inner is None or (inner_rows, inner_columns) == (rows, hidden)) and (not grouped or found[17:] == (1, groups + 1, groups + 1))):
            check_stream().gated_gemm_gradient(pre_gradient.buffer, stride, _buffer(inner), inner_stride, activation, output_gradient.buffer, width,
                                               a_stride, B.buffer, hidden, b_row_stride, b_stride, pre.buffer, pre_stride, _buffer(offsets), groups,
                                               rows)
            return pre_gradient
    _needed(name, pre_gradient=pre_gradient, output_gradient=output_gradient, B=B, pre=pre)
    _floating(name, pre_gradient, inner, output_gradient, B, pre)
    _indexes(name, pre_gradient, offsets=offsets)
    rows, columns, stride = _rows(name, "pre gradient", pre_gradient)
    a_rows, width, a_stride = _rows(name, "output gradient", output_gradient)
    pre_rows, pre_columns, pre_stride = _rows(name, "pre", pre)
    groups, b_rows, hidden, b_row_stride, b_stride = _weights(name, "B", B, offsets)
    if b_rows != width:
        raise TensorError(f"{name}: {width} columns of the output's gradient and {b_rows} by {hidden} of B do not go together")
    if (rows, columns) != (pre_rows, pre_columns) or (rows, columns) != (a_rows, 2 * hidden):
        raise TensorError(f"{name}: pre and its gradient must be {a_rows} by {2 * hidden}, got {list(pre.shape())} and {list(pre_gradient.shape())}")
    inner_stride = 0
    if inner is not None:
        inner_rows, inner_columns, inner_stride = _rows(name, "inner", inner)
        if (inner_rows, inner_columns) != (rows, hidden):
            raise TensorError(f"{name}: inner must be {rows} by {hidden}, got {list(inner.shape())}")
    if offsets is not None:
        _packed(name, "offsets", offsets, [groups + 1])
    check_stream().gated_gemm_gradient(pre_gradient.buffer, stride, _buffer(inner), inner_stride, activation, output_gradient.buffer, width, a_stride,
                                       B.buffer, hidden, b_row_stride, b_stride, pre.buffer, pre_stride, _buffer(offsets), groups, rows)
    return pre_gradient


# ---------------------------------------------------------------- a token's results

def combine_experts(output: Tensor, rows: Tensor, weights: Tensor, slots: Tensor) -> Tensor:
    """output[t] = sum over j of weights[t, j] * rows[slots[t, j]]; slots outside the rows are left out.  ``weights`` None
    means ones."""
    name = "combine-experts"
    found = _operands("mmpi", (output, rows, weights, slots))
    if found is not None:
        n, width, stride, count, columns, rows_stride = found[:6]
        of_choice = found[9:]
        if (columns == width and of_choice[0] == 2 and of_choice[1] == n * of_choice[2] and
                (weights is None or found[6:9] == of_choice)):
            check_stream().combine_experts(output.buffer, stride, rows.buffer, count, rows_stride, _buffer(weights), slots.buffer, n,
                                           of_choice[2], width)
            return output
    _needed(name, output=output, rows=rows, slots=slots)
    _floating(name, output, rows, weights)
    _indexes(name, output, slots=slots)
    n, width, stride = _rows(name, "output", output)
    count, columns, rows_stride = _rows(name, "rows", rows)
    n_chosen = int(slots.shape()[-1])
    _packed(name, "slots", slots, [n, n_chosen])
    _packed(name, "weights", weights, [n, n_chosen])
    if columns != width:
        raise TensorError(f"{name}: rows of {columns} and results of {width}")
    check_stream().combine_experts(output.buffer, stride, rows.buffer, count, rows_stride, _buffer(weights), slots.buffer, n, n_chosen,
                                   width)
    return output


def combine_experts_gradient(rows_gradient: Tensor, weights_gradient: Tensor, output_gradient: Tensor, rows: Tensor,
                             weights: Tensor, slots: Tensor) -> None:
    """rows-gradient[slots[t, j]] = weights[t, j] * output-gradient[t] (rows that no slot names are left as they are) and
    weights-gradient[t, j] = output-gradient[t] . rows[slots[t, j]].  Either may be None."""
    name = "combine-experts-gradient"
    found = _operands("mmmppi", (output_gradient, rows_gradient, rows, weights_gradient, weights, slots))
    if found is not None:
        n, width, stride, to_count, to_columns, to_stride, count, columns, rows_stride = found[:9]
        of_choice = found[15:]
        if (of_choice[0] == 2 and of_choice[1] == n * of_choice[2] and (rows_gradient is None or to_columns == width) and
                (columns == width if rows is not None else weights_gradient is None) and (not to_count or not count or to_count == count) and
                (weights_gradient is None or found[9:12] == of_choice) and (weights is None or found[12:15] == of_choice)):
            check_stream().combine_experts_gradient(_buffer(rows_gradient), to_stride or width, _buffer(weights_gradient), output_gradient.buffer,
                                                    stride, _buffer(rows), to_count or count, rows_stride or width, _buffer(weights),
                                                    slots.buffer, n, of_choice[2], width)
            return
    _needed(name, output_gradient=output_gradient, slots=slots)
    _floating(name, output_gradient, rows_gradient, weights_gradient, rows, weights)
    _indexes(name, output_gradient, slots=slots)
    n, width, stride = _rows(name, "output gradient", output_gradient)
    n_chosen = int(slots.shape()[-1])
    _packed(name, "slots", slots, [n, n_chosen])
    _packed(name, "weights", weights, [n, n_chosen])
    _packed(name, "weights gradient", weights_gradient, [n, n_chosen])
    if rows is None and weights_gradient is not None:
        raise TensorError(f"{name}: the rows are needed for the weights' gradient")
    count, to_stride, rows_stride = 0, width, width
    for what, t in (("rows gradient", rows_gradient), ("rows", rows)):
        if t is None:
            continue
        of, columns, row_stride = _rows(name, what, t)
        if columns != width or (count and of != count):
            raise TensorError(f"{name}: {what} {list(t.shape())} does not go with results of {width}")
        count = of
        if t is rows_gradient:
            to_stride = row_stride
        else:
            rows_stride = row_stride
    check_stream().combine_experts_gradient(_buffer(rows_gradient), to_stride, _buffer(weights_gradient), output_gradient.buffer, stride,
                                            _buffer(rows), count, rows_stride, _buffer(weights), slots.buffer, n, n_chosen, width)


# ---------------------------------------------------------------- the layers

def _norms(parameters, which):
    return {k: v[which] for k, v in parameters.items() if k in _OF_COLUMNS + ("gate",) and v.get(which) is not None}


class GatedBlock:
    """A residual gated feed-forward block, as it stands between two others:

        x = N_pre(residual)                             (what entered: norm_residual of the block before, or of this one)
        y = second * (f(gate) * up),  [gate up] = first * x
        output, normalized = norm_residual(y, residual)

    in the manner of :class:`ExpertBlock`: ``parameters`` is a dict of {"buffer", "gradient"} tensors, "first" [2 * hidden, width] with the
    gate's projection above the other's, "second" [width, hidden] and those of the norms.  Gradients are overwritten.  With ``training``
    false there is no backward pass, and what it would need is not kept."""

    def __init__(self, tokens: int, width: int, hidden: int, descriptor: dict = None, datatype: str = None, activation: str = "swish",
                 training: bool = True):
        _gate("gated-block", activation)
        self.descriptor = descriptor or norm_descriptor()
        self.activation = activation
        new = lambda shape: ct.new_tensor(shape, datatype=datatype)
        self.inner, self.combined = new([tokens, hidden]), new([tokens, width])
        self.statistics, self.pre, self.combined_gradient = ((new([4, tokens]), new([tokens, 2 * hidden]), new([tokens, width])) if training
                                                             else (None, None, None))

    def forward(self, parameters: dict, x: Tensor, residual: Tensor, output: Tensor, normalized: Tensor):
        gated_gemm(self.inner, self.pre, x, parameters["first"]["buffer"], activation=self.activation)
        ct.gemm(self.combined, False, True, 1.0, self.inner, parameters["second"]["buffer"], 0.0)
        return norm_residual(output, normalized, self.statistics, self.combined, residual, _norms(parameters, "buffer"), self.descriptor)

    def backward(self, parameters: dict, x: Tensor, output: Tensor, x_gradient: Tensor, residual_gradient: Tensor,
                 output_gradient: Tensor, normalized_gradient: Tensor):
        """The gradients of x and of the residual and of every parameter that has one, from those of the results, once to a forward pass:
        what that kept is overwritten.  A parameter whose "gradient" is None or absent is held as it is."""
        if self.pre is None:
            raise TensorError("gated-block: there is no backward pass of a block that is not for training")
        first, second = (parameters[k].get("gradient") for k in ("first", "second"))
        norm_residual_gradient(self.combined_gradient, residual_gradient, _norms(parameters, "gradient"), output_gradient,
                               normalized_gradient, self.combined, output, self.statistics, _norms(parameters, "buffer"), self.descriptor)
        if second is not None:
            ct.gemm(second, True, False, 1.0, self.combined_gradient, self.inner, 0.0)
        gated_gemm_gradient(self.pre, None, self.combined_gradient, parameters["second"]["buffer"], self.pre, activation=self.activation)
        if first is not None:
            ct.gemm(first, True, False, 1.0, self.pre, x, 0.0)
        ct.gemm(x_gradient, False, False, 1.0, self.pre, parameters["first"]["buffer"], 0.0)
        return x_gradient, residual_gradient


class ExpertBlock:
    """A residual feed-forward block of experts, as it stands between two others:

        x = N_pre(residual)                             (what entered: norm_residual of the block before, or of this one)
        route x * router^T;  y = experts' second products of relu(first products of x)
        output, normalized = norm_residual(y, residual)

    in the manner of :mod:`cortex_amd.nn_layers`: ``parameters`` is a dict of {"buffer", "gradient"} tensors, "router"
    [experts, width], "first" [experts, hidden, width], "second" [experts, width, hidden] and those of the norms
    ("post-scale", "pre-scale", ..., "gate").  Gradients are overwritten, one block to a batch.

    With ``gated``, one of :data:`GATES`, the experts are gated: "first" is [experts, 2 * hidden, width], the gates' projection above the
    others', and the inner rows are f(gate) * up in place of the relu; a backward pass then overwrites what the forward pass kept."""

    def __init__(self, tokens: int, width: int, hidden: int, n_experts: int, n_chosen: int, descriptor: dict = None,
                 datatype: str = None, renormalize: bool = True, gated: str = None):
        if gated is not None:
            _gate("expert-block", gated)
        self.descriptor = descriptor or norm_descriptor()
        self.renormalize = renormalize
        self.gated = gated
        rows = tokens * n_chosen
        new = lambda shape, kind=datatype: ct.new_tensor(shape, datatype=kind)
        self.logits, self.logits_gradient = new([tokens, n_experts]), new([tokens, n_experts])
        self.weights, self.weights_gradient = new([tokens, n_chosen]), new([tokens, n_chosen])
        self.experts, self.slots = new([tokens, n_chosen], "int"), new([tokens, n_chosen], "int")
        self.offsets, self.tokens = new([n_experts + 1], "int"), new([rows], "int")
        # a row to each assignment, in order of experts
        self.inner = new([rows, hidden])
        self.pre, self.inner_gradient = (None, new([rows, hidden])) if gated is None else (new([rows, 2 * hidden]), None)
        self.outer, self.outer_gradient = new([rows, width]), new([rows, width])
        self.combined, self.combined_gradient = new([tokens, width]), new([tokens, width])
        self.statistics = new([4, tokens])

    def forward(self, parameters: dict, x: Tensor, residual: Tensor, output: Tensor, normalized: Tensor):
        p = {k: v["buffer"] for k, v in parameters.items()}
        ct.gemm(self.logits, False, True, 1.0, x, p["router"], 0.0)
        route_experts(self.experts, self.weights, self.offsets, self.tokens, self.slots, self.logits, renormalize=self.renormalize)
        if self.gated is not None:
            gated_gemm(self.inner, self.pre, x, p["first"], self.offsets, self.tokens, activation=self.gated)
        else:
            grouped_gemm(self.inner, True, 1.0, x, p["first"], 0.0, self.offsets, index=self.tokens)
            ct.binary_op(self.inner, 1.0, self.inner, 1.0, 0, "max")
        grouped_gemm(self.outer, True, 1.0, self.inner, p["second"], 0.0, self.offsets)
        combine_experts(self.combined, self.outer, self.weights, self.slots)
        return norm_residual(output, normalized, self.statistics, self.combined, residual, _norms(parameters, "buffer"),
                             self.descriptor)

    def backward(self, parameters: dict, x: Tensor, output: Tensor, x_gradient: Tensor, residual_gradient: Tensor,
                 output_gradient: Tensor, normalized_gradient: Tensor):
        """The gradients of x and of the residual and of every parameter that has one, from those of the results.  A parameter whose
        "gradient" is None or absent is held as it is: nothing is formed for it alone."""
        p = {k: v["buffer"] for k, v in parameters.items()}
        router, first, second = (parameters[k].get("gradient") for k in ("router", "first", "second"))
        norm_residual_gradient(self.combined_gradient, residual_gradient, _norms(parameters, "gradient"), output_gradient,
                               normalized_gradient, self.combined, output, self.statistics, _norms(parameters, "buffer"),
                               self.descriptor)
        combine_experts_gradient(self.outer_gradient, self.weights_gradient, self.combined_gradient, self.outer, self.weights,
                                 self.slots)
        if second is not None:
            grouped_gemm_weights(second, 1.0, self.outer_gradient, self.inner, 0.0, self.offsets)
        if self.gated is not None:
            inner_gradient = gated_gemm_gradient(self.pre, None, self.outer_gradient, p["second"], self.pre, self.offsets, activation=self.gated)
        else:
            inner_gradient = grouped_gemm(self.inner_gradient, False, 1.0, self.outer_gradient, p["second"], 0.0, self.offsets)
            ct.activation_gradient(inner_gradient, inner_gradient, self.inner, "relu")
        if first is not None:
            grouped_gemm_weights(first, 1.0, inner_gradient, x, 0.0, self.offsets, b_index=self.tokens)
        # the gradient of x: of its rows among the experts, and of the router's
        grouped_gemm(self.outer_gradient, False, 1.0, inner_gradient, p["first"], 0.0, self.offsets)
        combine_experts(x_gradient, self.outer_gradient, None, self.slots)
        route_experts_gradient(self.logits_gradient, self.weights_gradient, self.weights, self.experts, self.logits,
                               renormalize=self.renormalize)
        if router is not None:
            ct.gemm(router, True, False, 1.0, self.logits_gradient, x, 0.0)
        ct.gemm(x_gradient, False, False, 1.0, self.logits_gradient, p["router"], 1.0)
        return x_gradient, residual_gradient
