"""What is measured of the operators that gated feed-forward blocks are computed with and that the matrices of a network are
trained with: the gated product (both projections of a row, the activation and the product of the two in one kernel) with its
backward pass, dense and by expert; the orthogonalisation of a matrix by Newton-Schulz products; and the optimizer step that
is made of it.

A case is a dict of plain values.  ``prepare`` makes the tensors that a program has in hand before the call, from a seed.
``run`` is one pass: where ``own`` is false in elementary operations of torch, where it is true through this library's entry
points on the same memory.  ``exact`` states the results once more in 64 bits.  Sizes are generic, or those of the layers on
digits that this library's own tests have.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TORCH = {"float": torch.float32, "double": torch.float64}
_SIZE = {"float": 4, "double": 8}


# ------------------------------------------------------------------------------------------------- the cases

def listed() -> list:
    return [
        # One token through a small block while a model answers: latency and the reading of the weights.
        {"name": "gated_one_token", "kind": "gated", "tokens": 1, "width": 1024, "hidden": 2816, "experts": 1, "chosen": 1,
         "activation": "swish", "backward": False, "datatype": "float"},
        # Sixteen sequences that answer at once, a large block: the reading of the weights.
        {"name": "gated_decode", "kind": "gated", "tokens": 16, "width": 4096, "hidden": 8192, "experts": 1, "chosen": 1,
         "activation": "swish", "backward": False, "datatype": "float"},
        # A training step of a dense block, all gradients.
        {"name": "gated_train", "kind": "gated", "tokens": 8192, "width": 1024, "hidden": 2816, "experts": 1, "chosen": 1,
         "activation": "swish", "backward": True, "datatype": "float"},
        # The same, of a wide one: the largest.
        {"name": "gated_train_wide", "kind": "gated", "tokens": 16384, "width": 2048, "hidden": 5632, "experts": 1, "chosen": 1,
         "activation": "swish", "backward": True, "datatype": "float"},
        # A training step of a block of experts, two of sixteen for each token.
        {"name": "gated_experts", "kind": "gated", "tokens": 4096, "width": 1024, "hidden": 1408, "experts": 16, "chosen": 2,
         "activation": "gelu", "backward": True, "datatype": "float"},
        # Odd sizes in double, as gradients are checked.
        {"name": "gated_double", "kind": "gated", "tokens": 509, "width": 301, "hidden": 517, "experts": 1, "chosen": 1,
         "activation": "logistic", "backward": True, "datatype": "double"},
        # An update of many matrices of one odd shape, taller than wide.
        {"name": "orthogonal_odd", "kind": "orthogonal", "rows": 1531, "columns": 517, "count": 6, "datatype": "float"},
        # A large matrix by itself.
        {"name": "orthogonal_large", "kind": "orthogonal", "rows": 4096, "columns": 8192, "count": 1, "datatype": "float"},
        # The first layer of a small network on digits: latency.
        {"name": "muon_digits", "kind": "muon", "rows": 128, "columns": 784, "count": 1, "nesterov": True, "decay": 0.0,
         "datatype": "float"},
        # One projection of a small block.
        {"name": "muon_square", "kind": "muon", "rows": 1024, "columns": 1024, "count": 1, "nesterov": True, "decay": 0.1,
         "datatype": "float"},
        # The matrices of sixteen experts in one step.
        {"name": "muon_experts", "kind": "muon", "rows": 2816, "columns": 1024, "count": 16, "nesterov": True, "decay": 0.1,
         "datatype": "float"},
        # In double, odd sizes.
        {"name": "muon_double", "kind": "muon", "rows": 301, "columns": 517, "count": 5, "nesterov": False, "decay": 0.01,
         "datatype": "double"},
    ]


def _log_int(rng, low: int, high: int) -> int:
    """A whole number in [low, high], even over its logarithm; powers of two are no likelier than others."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _type(rng) -> str:
    return rng.choice(["float", "float", "float", "double"])


def _draw_gated(rng):
    while True:
        experts = rng.choice([1, 1, 1, _log_int(rng, 2, 32)])
        case = {"tokens": _log_int(rng, 1, 16384), "width": _log_int(rng, 16, 4096), "hidden": _log_int(rng, 16, 8192),
                "experts": experts, "chosen": min(experts, rng.choice([1, 2, 2, 4]))}
        datatype = _type(rng)
        values = case["width"] * case["hidden"]
        if case["tokens"] * case["chosen"] * values <= 1 << (36 if datatype == "float" else 32) and experts * values <= 1 << 26:
            return dict(case, activation=rng.choice(["swish", "swish", "gelu", "logistic", "relu", "tanh"]),
                        backward=rng.random() < 0.6, datatype=datatype)


def _draw_matrices(rng):
    while True:
        case = {"rows": _log_int(rng, 4, 8192), "columns": _log_int(rng, 4, 8192), "count": rng.choice([1, 1, 1, _log_int(rng, 2, 32)])}
        datatype = _type(rng)
        small, large = sorted((case["rows"], case["columns"]))
        if case["count"] * small * small * large <= 1 << (36 if datatype == "float" else 31):
            return dict(case, datatype=datatype)


def _draw_muon(rng):
    return dict(_draw_matrices(rng), nesterov=rng.random() < 0.7, decay=rng.choice([0.0, 0.01, 0.1]))


_DRAW = {"gated": _draw_gated, "orthogonal": _draw_matrices, "muon": _draw_muon}


def draw(rng) -> dict:
    kind = rng.choice(sorted(_DRAW))
    return dict(_DRAW[kind](rng), kind=kind)


# ------------------------------------------------------------------------------------------------- shared pieces

_DEVICE = None


class _State:
    """What a pass works on: torch tensors and, for the library's calls, its views of the same memory."""

    def __init__(self, case: dict, seed: int):
        self.case = case
        self.dtype = _TORCH[case["datatype"]]
        self.generator = torch.Generator(device="cuda").manual_seed(seed)
        self.host = np.random.default_rng(seed)
        self._library = None

    def normal(self, *shape, mean=0.0, std=1.0):
        return torch.empty(shape, device="cuda", dtype=self.dtype).normal_(mean, std, generator=self.generator)

    def empty(self, *shape, dtype=None):
        return torch.empty(shape, device="cuda", dtype=dtype or self.dtype)

    def indexes(self, array):
        return torch.from_numpy(np.ascontiguousarray(array, dtype=np.int32)).cuda()

    def view(self, t: torch.Tensor):
        """The library's tensor over a torch tensor, which lives as long as the view."""
        from cortex_amd import dimensions, driver, tensor
        global _DEVICE
        if _DEVICE is None:
            _DEVICE = driver.HipDriver().default_device()
        names = {torch.float32: "float", torch.float64: "double", torch.int32: "int"}
        buffer = driver.DeviceBuffer(_DEVICE, t.data_ptr(), t.numel(), names[t.dtype])
        buffer.storage = t
        return tensor.Tensor(_DEVICE, dimensions.dimensions(list(t.shape)), buffer)

    def bind(self):
        """The stream that the calls are made on: torch's own."""
        from cortex_amd import driver, tensor
        if self._library is None:
            self._library = driver.HipStream(self.view(self.empty(1)).device, torch.cuda.current_stream().cuda_stream or None)
        return tensor.tensor_context(self._library, self.case["datatype"])


def prepare(case: dict, seed: int):
    s = _State(case, seed)
    _PREPARE[case["kind"]](s)
    return s


def run(state):
    kind = state.case["kind"]
    if not own:
        return _PLAIN[kind](state)
    with state.bind():
        return _OWN[kind](state)


def work(case: dict) -> dict:
    values, others, flops = _WORK[case["kind"]](case)
    return {"bytes": values * _SIZE[case["datatype"]] + others, "flops": flops}


def exact(case: dict, seed: int):
    return _EXACT[case["kind"]](prepare(case, seed))


# ------------------------------------------------------------------------------------------------- the gated product

def _prepare_gated(s):
    c = s.case
    n, k, e, width, hidden = c["tokens"], c["chosen"], c["experts"], c["width"], c["hidden"]
    rows = n * k
    s.input = s.normal(n, width)
    # gate and up projection one behind the other, and the projection back
    groups = (e,) if e > 1 else ()
    s.first = s.normal(*groups, 2 * hidden, width, std=1.0 / math.sqrt(width))
    s.second = s.normal(*groups, width, hidden, std=1.0 / math.sqrt(hidden))
    s.sizes, s.offsets, s.tokens = [rows], None, None
    if e > 1:
        # how many rows an expert has is uneven; which token a row is of
        liked = np.exp(s.host.normal(0.0, 0.5, e))
        sizes = s.host.multinomial(rows, liked / liked.sum())
        s.sizes, s.offsets = sizes.tolist(), s.indexes(np.concatenate([[0], np.cumsum(sizes)]))
        s.tokens = s.indexes(s.host.permutation(rows) // k)
    s.inner, s.result = s.empty(rows, hidden), s.empty(rows, width)
    if c["backward"]:
        s.result_gradient = s.normal(rows, width, std=1e-2)
        s.pre, s.pre_gradient = s.empty(rows, 2 * hidden), s.empty(rows, 2 * hidden)
        s.rows_gradient = s.empty(rows, width)
        s.first_gradient, s.second_gradient = torch.empty_like(s.first), torch.empty_like(s.second)


def _plain_activation(g, kind):
    """The activation and its derivative."""
    if kind == "swish":
        p = 1.0 / (1.0 + torch.exp(-g))
        return g * p, p * (1.0 + g * (1.0 - p))
    if kind == "gelu":
        share = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * share, share + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    if kind == "logistic":
        p = 1.0 / (1.0 + torch.exp(-g))
        return p, p * (1.0 - p)
    if kind == "tanh":
        t = torch.tanh(g)
        return t, 1.0 - t * t
    return torch.clamp(g, min=0.0), (g > 0).to(g.dtype)


def _plain_gated(s):
    c = s.case
    hidden, e = c["hidden"], c["experts"]
    if e > 1:
        # the groups side by side, each as long as the longest
        row = torch.arange(c["tokens"] * c["chosen"], device="cuda")
        group = torch.searchsorted(s.offsets[1:].contiguous(), row.to(torch.int32), right=True)
        place, most = row - s.offsets[group], max(s.sizes)
        spread = lambda t: t.new_zeros(e, most, t.shape[1]).index_put((group, place), t)
        gather = lambda t: t[group, place]
        taken = spread(s.input[s.tokens.long()])
    else:
        spread = gather = lambda t: t
        taken = s.input
    turned = lambda t: t.transpose(-1, -2).contiguous()
    pre = torch.matmul(taken, turned(s.first))
    act, slope = _plain_activation(pre[..., :hidden], c["activation"])
    up = pre[..., hidden:]
    inner = act * up
    result = {"inner": gather(inner), "result": gather(torch.matmul(inner, turned(s.second)))}
    if c["backward"]:
        gradient = spread(s.result_gradient)
        inner_gradient = torch.matmul(gradient, s.second)
        pre_gradient = torch.cat([inner_gradient * up * slope, inner_gradient * act], dim=-1)
        result["pre_gradient"] = gather(pre_gradient)
        result["rows_gradient"] = gather(torch.matmul(pre_gradient, s.first))
        result["first_gradient"] = torch.matmul(turned(pre_gradient), taken)
        result["second_gradient"] = torch.matmul(turned(gradient), inner)
    return result


def _own_gated(s):
    from cortex_amd import blocks, tensor
    c = s.case
    if not hasattr(s, "views"):
        s.views = [s.view(t) for t in (s.inner, s.result, s.input, s.first, s.second)]
        s.groups = [s.view(t) for t in (s.offsets, s.tokens)] if c["experts"] > 1 else [None, None]
        if c["backward"]:
            s.gradient_views = [s.view(t) for t in (s.pre, s.pre_gradient, s.result_gradient, s.rows_gradient, s.first_gradient,
                                                    s.second_gradient)]
    inner, result, input, first, second = s.views
    offsets, tokens = s.groups
    pre = s.gradient_views[0] if c["backward"] else None
    blocks.gated_gemm(inner, pre, input, first, offsets, tokens, activation=c["activation"])
    if offsets is not None:
        blocks.grouped_gemm(result, True, 1.0, inner, second, 0.0, offsets)
    else:
        tensor.gemm(result, False, True, 1.0, inner, second, 0.0)
    found = {"inner": s.inner, "result": s.result}
    if not c["backward"]:
        return found
    pre, pre_gradient, result_gradient, rows_gradient, first_gradient, second_gradient = s.gradient_views
    blocks.gated_gemm_gradient(pre_gradient, None, result_gradient, second, pre, offsets, activation=c["activation"])
    if offsets is not None:
        blocks.grouped_gemm(rows_gradient, False, 1.0, pre_gradient, first, 0.0, offsets)
        blocks.grouped_gemm_weights(first_gradient, 1.0, pre_gradient, input, 0.0, offsets, b_index=tokens)
        blocks.grouped_gemm_weights(second_gradient, 1.0, result_gradient, inner, 0.0, offsets)
    else:
        tensor.gemm(rows_gradient, False, False, 1.0, pre_gradient, first, 0.0)
        tensor.gemm(first_gradient, True, False, 1.0, pre_gradient, input, 0.0)
        tensor.gemm(second_gradient, True, False, 1.0, result_gradient, inner, 0.0)
    return dict(found, pre_gradient=s.pre_gradient, rows_gradient=s.rows_gradient, first_gradient=s.first_gradient,
                second_gradient=s.second_gradient)


def _work_gated(c):
    n, k, e, width, hidden = c["tokens"], c["chosen"], c["experts"], c["width"], c["hidden"]
    rows = n * k
    weights = min(e, rows) * 3 * width * hidden
    values, flops = n * width + rows * hidden + rows * width + weights, 6 * rows * width * hidden
    if c["backward"]:
        values, flops = values + 2 * rows * width + 2 * rows * hidden + 3 * e * width * hidden, 3 * flops
    return values, 4 * (rows + e if e > 1 else 0), flops


def _exact_gated(s):
    c = s.case
    hidden, kind, at, parts = c["hidden"], c["activation"], 0, []
    rows = s.input.double() if c["experts"] == 1 else s.input.double()[s.tokens.long()]
    first, second = (t.double().reshape(c["experts"], *t.shape[-2:]) for t in (s.first, s.second))
    for i, size in enumerate(s.sizes):
        x = rows[at:at + size]
        gate, up = x @ first[i, :hidden].t(), x @ first[i, hidden:].t()
        if kind == "swish":
            act = gate * torch.sigmoid(gate)
            slope = torch.sigmoid(gate) + act * torch.sigmoid(-gate)
        elif kind == "gelu":
            normal = torch.special.ndtr(gate)
            act, slope = gate * normal, normal + gate * torch.exp(-gate ** 2 / 2) / math.sqrt(2 * math.pi)
        elif kind == "logistic":
            act, slope = torch.sigmoid(gate), torch.sigmoid(gate) * torch.sigmoid(-gate)
        elif kind == "tanh":
            act, slope = torch.tanh(gate), 1 / torch.cosh(gate) ** 2
        else:
            act, slope = gate.where(gate > 0, torch.zeros_like(gate)), torch.heaviside(gate, torch.zeros_like(gate))
        inner = act * up
        part = {"inner": inner, "result": inner @ second[i].t()}
        if c["backward"]:
            dy = s.result_gradient[at:at + size].double()
            back = dy @ second[i]
            gradient = torch.cat([back * up * slope, back * act], 1)
            part.update(pre_gradient=gradient, rows_gradient=gradient @ first[i], first_gradient=(gradient.t() @ x)[None],
                        second_gradient=(dy.t() @ inner)[None])
        parts.append(part)
        at += size
    found = {name: torch.cat([part[name] for part in parts]) for name in parts[0]}
    if c["backward"]:
        found["first_gradient"] = found["first_gradient"].reshape(s.first.shape)
        found["second_gradient"] = found["second_gradient"].reshape(s.second.shape)
    return found


# ------------------------------------------------------------------------------------------------- matrices made orthogonal

_STEPS, _EPSILON = 5, 1e-7
_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_ALPHA, _MOMENTUM, _BATCH = 0.02, 0.95, 64


def _gradient(s):
    """As the gradients of matrices are: a few directions carry most of it, the rest is noise."""
    c = s.case
    rank = max(1, min(c["rows"], c["columns"]) // 8)
    left, right = s.normal(c["count"], c["rows"], rank), s.normal(c["count"], rank, c["columns"])
    left *= torch.arange(1, rank + 1, device="cuda", dtype=s.dtype).rsqrt()
    return torch.bmm(left, right) * (1e-3 / math.sqrt(rank)) + s.normal(c["count"], c["rows"], c["columns"], std=2e-4)


def _prepare_orthogonal(s):
    s.input = _gradient(s)
    s.output = torch.empty_like(s.input)


def _prepare_muon(s):
    # sums over a batch; what they had come to before; the matrices
    s.gradient, s.momentum_before = _gradient(s) * _BATCH, _gradient(s) * 8
    s.parameters_before = s.normal(*s.gradient.shape, std=1.0 / math.sqrt(s.case["columns"]))
    s.momentum, s.parameters = torch.empty_like(s.gradient), torch.empty_like(s.gradient)


def _plain_orthogonal_of(matrix):
    tall = matrix.shape[-2] > matrix.shape[-1]
    x = matrix.transpose(-1, -2).contiguous() if tall else matrix
    x = x / ((x * x).sum(dim=(-2, -1), keepdim=True).sqrt() + _EPSILON)
    a, b, c = _COEFFICIENTS
    for _ in range(_STEPS):
        square = torch.bmm(x, x.transpose(-1, -2).contiguous())
        x = a * x + torch.bmm(b * square + c * torch.bmm(square, square), x)
    return x.transpose(-1, -2).contiguous() if tall else x


def _plain_orthogonal(s):
    return {"output": _plain_orthogonal_of(s.input)}


def _plain_muon(s):
    c = s.case
    gradient = s.gradient * (1.0 / _BATCH)
    momentum = _MOMENTUM * s.momentum_before + gradient
    update = _plain_orthogonal_of(gradient + _MOMENTUM * momentum if c["nesterov"] else momentum)
    rate = _ALPHA * math.sqrt(max(1.0, c["rows"] / c["columns"]))
    return {"parameters": s.parameters_before * (1.0 - _ALPHA * c["decay"]) - rate * update, "momentum": momentum}


def _own_orthogonal(s):
    from cortex_amd import optimize, tensor
    if not hasattr(s, "views"):
        s.views = [s.view(t) for t in (s.output, s.input)]
        s.backend = optimize.Backend(tensor.check_stream(), s.case["datatype"])
        s.workspace = optimize.orthogonalize_workspace(s.backend, s.views[1])
    optimize.orthogonalize(s.backend, *s.views, steps=_STEPS, coefficients=_COEFFICIENTS, epsilon=_EPSILON, workspace=s.workspace)
    return {"output": s.output}


def _own_muon(s):
    from cortex_amd import optimize, tensor
    c = s.case
    if not hasattr(s, "views"):
        s.views = [s.view(t) for t in (s.momentum, s.gradient, s.parameters)]
        s.optimizer = optimize.create_optimizer(
            optimize.Backend(tensor.check_stream(), c["datatype"]),
            optimize.muon(alpha=_ALPHA, momentum=_MOMENTUM, nesterov=c["nesterov"], steps=_STEPS, coefficients=_COEFFICIENTS,
                          epsilon=_EPSILON, **{"weight-decay": c["decay"]}))
    # the step is made in place; what it began with is kept, as a program does that may have to take a step back
    s.momentum.copy_(s.momentum_before)
    s.parameters.copy_(s.parameters_before)
    momentum, gradient, parameters = s.views
    s.optimizer.batch_update().compute_parameters({"momentum-vals": momentum}, 1.0 / _BATCH, 0, gradient, parameters)
    return {"parameters": s.parameters, "momentum": s.momentum}


def _flops_orthogonal(c):
    """A product of a matrix by its transpose is symmetric, and so is that one's square: half of each is computed."""
    small, large = sorted((c["rows"], c["columns"]))
    return c["count"] * _STEPS * (small * (small + 1) * large + small * small * (small + 1) + 2 * small * small * large)


def _work_orthogonal(c):
    return 2 * c["count"] * c["rows"] * c["columns"], 0, _flops_orthogonal(c)


def _work_muon(c):
    return 5 * c["count"] * c["rows"] * c["columns"], 0, _flops_orthogonal(c)


def _exact_orthogonal_of(g):
    """With the smaller Gram matrix, of the rows or of the columns, beside the matrix as it lies."""
    x = g / (torch.linalg.vector_norm(g) + _EPSILON)
    a, b, c = _COEFFICIENTS
    rows, columns = x.shape
    eye = torch.eye(min(rows, columns), device=x.device, dtype=x.dtype)
    for _ in range(_STEPS):
        gram = x @ x.t() if rows <= columns else x.t() @ x
        factor = a * eye + gram @ (b * eye + c * gram)
        x = factor @ x if rows <= columns else x @ factor
    return x


def _exact_orthogonal(s):
    return {"output": torch.stack([_exact_orthogonal_of(g) for g in s.input.double()])}


def _exact_muon(s):
    c = s.case
    gradient, before = s.gradient.double() / _BATCH, s.momentum_before.double()
    momentum = before * _MOMENTUM + gradient
    looked_ahead = (before * _MOMENTUM + gradient) * _MOMENTUM + gradient if c["nesterov"] else momentum
    update = torch.stack([_exact_orthogonal_of(u) for u in looked_ahead])
    shrunk = s.parameters_before.double() * (1.0 - _ALPHA * c["decay"])
    return {"parameters": shrunk - update * (_ALPHA * max(1.0, c["rows"] / c["columns"]) ** 0.5), "momentum": momentum}


_PREPARE = {"gated": _prepare_gated, "orthogonal": _prepare_orthogonal, "muon": _prepare_muon}
_PLAIN = {"gated": _plain_gated, "orthogonal": _plain_orthogonal, "muon": _plain_muon}
_OWN = {"gated": _own_gated, "orthogonal": _own_orthogonal, "muon": _own_muon}
_WORK = {"gated": _work_gated, "orthogonal": _work_orthogonal, "muon": _work_muon}
_EXACT = {"gated": _exact_gated, "orthogonal": _exact_orthogonal, "muon": _exact_muon}
