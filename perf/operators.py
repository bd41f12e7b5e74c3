"""What is measured of the operators that a residual block of experts is trained and served with: the norms around a block
with its gate and residual, the choice of experts and the order of rows that follows from it, the products grouped by
expert, the sum of a token's results, and the norm of all gradients with their clipping.

A case is a dict of plain values.  ``prepare`` makes the tensors that a program has in hand before the call, from a seed.
``run`` is one pass: where ``own`` is false in elementary operations of torch, where it is true through this library's entry
points on the same memory.  ``exact`` states the results once more in 64 bits.  Sizes are generic.
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
        # One token on its way from one block to the next while a model answers: latency is everything.
        {"name": "norm_one_token", "kind": "norm", "rows": 1, "width": 4096, "post": "rms", "pre": "rms", "gate": "column",
         "biases": False, "backward": False, "datatype": "float"},
        # The same place in a training step, forward and backward.
        {"name": "norm_train", "kind": "norm", "rows": 16384, "width": 2048, "post": "rms", "pre": "rms", "gate": "column",
         "biases": False, "backward": True, "datatype": "float"},
        # Centered norms with biases and a gate for each row, rows of an odd length, in double.
        {"name": "norm_layer_double", "kind": "norm", "rows": 5003, "width": 1531, "post": "layer", "pre": "layer",
         "gate": "row", "biases": True, "backward": True, "datatype": "double"},
        # Sixteen sequences that answer at once, eight of 64 experts each.
        {"name": "route_decode", "kind": "route", "tokens": 16, "experts": 64, "chosen": 8, "renormalize": True,
         "masked": 0.0, "backward": False, "datatype": "float"},
        # The tokens of a training step; some experts are closed to some tokens.
        {"name": "route_train", "kind": "route", "tokens": 65536, "experts": 128, "chosen": 8, "renormalize": False,
         "masked": 0.1, "backward": True, "datatype": "float"},
        # A first product of experts for eight sequences that answer at once: the weights of the chosen experts are read.
        {"name": "products_decode", "kind": "products", "tokens": 8, "chosen": 2, "experts": 16, "inputs": 2048,
         "outputs": 4096, "skew": 0.5, "backward": False, "datatype": "float"},
        # The same product in a training step, with both gradients.
        {"name": "products_train", "kind": "products", "tokens": 8192, "chosen": 2, "experts": 16, "inputs": 1024,
         "outputs": 2048, "skew": 0.5, "backward": True, "datatype": "float"},
        # Odd sizes and uneven groups in double, as gradients are checked.
        {"name": "products_double", "kind": "products", "tokens": 1013, "chosen": 2, "experts": 7, "inputs": 301,
         "outputs": 517, "skew": 1.0, "backward": True, "datatype": "double"},
        # Results of experts brought together again: a few tokens, and a training step with its gradients.
        {"name": "combine_decode", "kind": "combine", "tokens": 16, "chosen": 2, "experts": 16, "width": 2048, "dropped": 0.0,
         "backward": False, "datatype": "float"},
        {"name": "combine_train", "kind": "combine", "tokens": 16384, "chosen": 4, "experts": 64, "width": 1000,
         "dropped": 0.02, "backward": True, "datatype": "float"},
        # The gradients of a small network on digits (784 -> 128 -> 10), and of a large one with many tensors.
        {"name": "clip_digits", "kind": "clip", "tensors": 4, "values": 101770, "most": 100352, "limit": 1.0,
         "datatype": "float"},
        {"name": "clip_large", "kind": "clip", "tensors": 300, "values": 200_000_000, "most": 16_777_216, "limit": 1.0,
         "datatype": "float"},
    ]


def _log_int(rng, low: int, high: int) -> int:
    """A whole number in [low, high], even over its logarithm; powers of two are no likelier than others."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _type(rng) -> str:
    return rng.choice(["float", "float", "float", "double"])


def _draw_norm(rng):
    post, pre = rng.choice([("rms", "rms"), ("layer", "layer"), ("none", "rms"), ("none", "layer"), ("rms", "none")])
    while True:
        case = {"rows": _log_int(rng, 1, 32768), "width": _log_int(rng, 16, 8192)}
        if case["rows"] * case["width"] <= 1 << 24:
            break
    return dict(case, post=post, pre=pre, gate=rng.choice(["none", "column", "row", "full"]), biases=rng.random() < 0.5,
                backward=rng.random() < 0.7, datatype=_type(rng))


def _draw_route(rng):
    experts = _log_int(rng, 2, 512)
    return {"tokens": _log_int(rng, 1, 65536 if experts <= 128 else 16384), "experts": experts,
            "chosen": min(experts, rng.choice([1, 2, 2, 4, 6, 8])), "renormalize": rng.random() < 0.5,
            "masked": rng.choice([0.0, 0.0, 0.1]), "backward": rng.random() < 0.5, "datatype": _type(rng)}


def _draw_products(rng):
    while True:
        experts = _log_int(rng, 2, 64)
        case = {"tokens": _log_int(rng, 1, 16384), "chosen": min(experts, rng.choice([1, 2, 2, 4])), "experts": experts,
                "inputs": _log_int(rng, 32, 4096), "outputs": _log_int(rng, 32, 4096)}
        datatype = _type(rng)
        values = case["inputs"] * case["outputs"]
        if case["tokens"] * case["chosen"] * values <= 1 << (35 if datatype == "float" else 33) and experts * values <= 1 << 27:
            return dict(case, skew=rng.choice([0.0, 0.5, 1.0]), backward=rng.random() < 0.6, datatype=datatype)


def _draw_combine(rng):
    while True:
        case = {"tokens": _log_int(rng, 1, 32768), "chosen": rng.choice([1, 2, 2, 4, 8]), "experts": _log_int(rng, 8, 256),
                "width": _log_int(rng, 32, 4096)}
        if case["tokens"] * case["chosen"] * case["width"] <= 1 << 26:
            return dict(case, dropped=rng.choice([0.0, 0.05]), backward=rng.random() < 0.6, datatype=_type(rng))


def _draw_clip(rng):
    tensors = _log_int(rng, 1, 500)
    values = _log_int(rng, max(1000, 4 * tensors), 1 << 26)
    return {"tensors": tensors, "values": values, "most": max(4, min(values, rng.choice([4, 8, 16]) * values // tensors)),
            "limit": rng.choice([1.0, 1.0, 1e6]), "datatype": _type(rng)}


_DRAW = {"norm": _draw_norm, "route": _draw_route, "products": _draw_products, "combine": _draw_combine, "clip": _draw_clip}


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


# ------------------------------------------------------------------------------------------------- norms, gate and residual

_EPSILON = 1e-5
_RESIDUAL_SCALE = 0.9


def _prepare_norm(s):
    c = s.case
    n, d = c["rows"], c["width"]
    s.input, s.residual = s.normal(n, d, mean=0.1), s.normal(n, d, std=2.0)
    s.parameters = {}
    for place in ("post", "pre"):
        if c[place] != "none":
            s.parameters[place + "-scale"] = s.normal(d, mean=1.0, std=0.1)
            if c["biases"]:
                s.parameters[place + "-bias"] = s.normal(d, std=0.1)
    if c["gate"] != "none":
        s.parameters["gate"] = s.normal(*{"column": (1, d), "row": (n, 1), "full": (n, d)}[c["gate"]], mean=0.5, std=0.3)
    s.output, s.normalized = s.empty(n, d), s.empty(n, d) if c["pre"] != "none" else None
    if c["backward"]:
        s.output_gradient = s.normal(n, d, std=1e-2)
        s.normalized_gradient = s.normal(n, d, std=1e-2) if c["pre"] != "none" else None
        s.input_gradient, s.residual_gradient = s.empty(n, d), s.empty(n, d)
        s.parameter_gradients = {k: torch.empty_like(v) for k, v in s.parameters.items()}
    s.statistics = s.empty(4, n) if c["backward"] else None


def _plain_norm_of(x, kind, scale, bias):
    if kind == "none":
        return x, None, None
    centered = x - x.mean(1, keepdim=True) if kind == "layer" else x
    rate = torch.rsqrt((centered * centered).mean(1, keepdim=True) + _EPSILON)
    hat = centered * rate
    out = hat * scale
    return (out if bias is None else out + bias), hat, rate


def _plain_norm_gradient(y, hat, rate, kind):
    out = y - hat * (y * hat).mean(1, keepdim=True)
    if kind == "layer":
        out = out - y.mean(1, keepdim=True)
    return out * rate


def _plain_norm(s):
    c, p = s.case, s.parameters
    block, input_hat, input_rate = _plain_norm_of(s.input, c["post"], p.get("post-scale"), p.get("post-bias"))
    gate = p.get("gate")
    output = _RESIDUAL_SCALE * s.residual + (block if gate is None else gate * block)
    normalized, hat, rate = _plain_norm_of(output, c["pre"], p.get("pre-scale"), p.get("pre-bias"))
    result = {"output": output}
    if c["pre"] != "none":
        result["normalized"] = normalized
    if not c["backward"]:
        return result
    total, gradients = s.output_gradient, {}
    if c["pre"] != "none":
        total = total + _plain_norm_gradient(s.normalized_gradient * p["pre-scale"], hat, rate, c["pre"])
        gradients["pre-scale"] = (s.normalized_gradient * hat).sum(0)
        gradients["pre-bias"] = s.normalized_gradient.sum(0)
    result["residual_gradient"] = _RESIDUAL_SCALE * total
    of_block = total
    if gate is not None:
        of_gate = total * block
        gradients["gate"] = {"column": lambda: of_gate.sum(0, keepdim=True), "row": lambda: of_gate.sum(1, keepdim=True),
                             "full": lambda: of_gate}[c["gate"]]()
        of_block = total * gate
    if c["post"] != "none":
        gradients["post-scale"] = (of_block * input_hat).sum(0)
        gradients["post-bias"] = of_block.sum(0)
        of_block = _plain_norm_gradient(of_block * p["post-scale"], input_hat, input_rate, c["post"])
    result["input_gradient"] = of_block
    result["parameters"] = {k: gradients[k] for k in p}
    return result


def _own_norm(s):
    from cortex_amd import blocks
    c = s.case
    if not hasattr(s, "views"):
        v = lambda t: None if t is None else s.view(t)
        of = lambda d: {k: v(t) for k, t in d.items()}
        s.views = (v(s.output), v(s.normalized), v(s.statistics), v(s.input), v(s.residual), of(s.parameters))
        s.descriptor = blocks.norm_descriptor(post=c["post"], pre=c["pre"], epsilon=_EPSILON, residual_scale=_RESIDUAL_SCALE)
        if c["backward"]:
            s.gradient_views = (v(s.input_gradient), v(s.residual_gradient), of(s.parameter_gradients), v(s.output_gradient),
                                v(s.normalized_gradient))
    output, normalized, statistics, input, residual, parameters = s.views
    blocks.norm_residual(output, normalized, statistics, input, residual, parameters, s.descriptor)
    result = {"output": s.output}
    if c["pre"] != "none":
        result["normalized"] = s.normalized
    if c["backward"]:
        blocks.norm_residual_gradient(*s.gradient_views, input, output, statistics, parameters, s.descriptor)
        result.update(residual_gradient=s.residual_gradient, input_gradient=s.input_gradient, parameters=s.parameter_gradients)
    return result


def _work_norm(c):
    n = c["rows"] * c["width"]
    pre = c["pre"] != "none"
    full = n if c["gate"] == "full" else 0
    values, flops = (3 + pre) * n + full, 10 * n
    if c["backward"]:
        values, flops = values + (5 + pre) * n + 2 * full, flops + 25 * n
    return values + 6 * c["width"], 0, flops


def _exact_norm(s):
    c = s.case
    leaf = lambda t: t.double().clone().requires_grad_(c["backward"])
    z, r, p = leaf(s.input), leaf(s.residual), {k: leaf(t) for k, t in s.parameters.items()}

    def norm(x, place):
        if c[place] == "none":
            return x
        if c[place] == "layer":
            x = x - x.sum(1, keepdim=True) / x.shape[1]
        x = x / ((x ** 2).sum(1, keepdim=True) / x.shape[1] + _EPSILON).sqrt() * p[place + "-scale"]
        return x + p[place + "-bias"] if c["biases"] else x

    output = norm(z, "post") * (p["gate"] if "gate" in p else 1.0) + _RESIDUAL_SCALE * r
    result = {"output": output.detach()}
    objective = (output * s.output_gradient.double()).sum() if c["backward"] else None
    if c["pre"] != "none":
        normalized = norm(output, "pre")
        result["normalized"] = normalized.detach()
        if c["backward"]:
            objective = objective + (normalized * s.normalized_gradient.double()).sum()
    if c["backward"]:
        objective.backward()
        result.update(residual_gradient=r.grad, input_gradient=z.grad, parameters={k: t.grad for k, t in p.items()})
    return result


# ------------------------------------------------------------------------------------------------- the choice of experts

def _prepare_route(s):
    c = s.case
    n, e, k = c["tokens"], c["experts"], c["chosen"]
    # experts differ in how much they are liked
    s.logits = s.normal(n, e) + s.normal(e, std=0.7)
    if c["masked"]:
        # some experts are closed to a token, one never is
        closed = torch.rand((n, e), device="cuda", generator=s.generator) < c["masked"]
        closed[:, 0] = False
        s.logits.masked_fill_(closed, -math.inf)
    s.weights = s.empty(n, k)
    i32 = torch.int32
    s.chosen, s.offsets = s.empty(n, k, dtype=i32), s.empty(e + 1, dtype=i32)
    s.order, s.slots = s.empty(n * k, dtype=i32), s.empty(n, k, dtype=i32)
    if c["backward"]:
        s.weights_gradient, s.logits_gradient = s.normal(n, k, std=1e-2), s.empty(n, e)


def _plain_route(s):
    c = s.case
    n, e, k = c["tokens"], c["experts"], c["chosen"]
    values, at = torch.sort(s.logits, dim=1, descending=True, stable=True)
    values, at = values[:, :k], at[:, :k]
    powers = torch.exp(values - values[:, :1])
    over = powers if c["renormalize"] else torch.exp(s.logits - values[:, :1])
    weights = powers / over.sum(1, keepdim=True)
    open_ = values > -math.inf
    chosen = torch.where(open_, at, e)   # what is closed comes after every expert
    order = torch.sort(chosen.reshape(-1), stable=True)[1]
    offsets = torch.searchsorted(chosen.reshape(-1)[order], torch.arange(e + 1, device="cuda"))
    places = torch.arange(n * k, device="cuda")
    slots = torch.empty_like(order)
    slots[order] = places
    slots = torch.where(open_.reshape(-1), slots, -1).reshape(n, k)
    tokens = torch.where(places < offsets[e], order // k, -1)
    i32 = torch.int32
    result = {"weights": weights, "experts": torch.where(open_, at, -1).to(i32), "offsets": offsets.to(i32),
              "tokens": tokens.to(i32), "slots": slots.to(i32)}
    if c["backward"]:
        common = (weights * s.weights_gradient).sum(1, keepdim=True)
        if c["renormalize"]:
            gradient = torch.zeros_like(s.logits)
        else:
            gradient = -common * torch.exp(s.logits - values[:, :1]) / over.sum(1, keepdim=True)
        taken = weights * (s.weights_gradient - common) if c["renormalize"] else weights * s.weights_gradient
        result["logits_gradient"] = gradient.scatter_add(1, at, taken)
    return result


def _own_route(s):
    from cortex_amd import blocks
    c = s.case
    if not hasattr(s, "views"):
        s.views = [s.view(t) for t in (s.chosen, s.weights, s.offsets, s.order, s.slots, s.logits)]
        if c["backward"]:
            s.gradient_views = [s.view(t) for t in (s.logits_gradient, s.weights_gradient)]
    experts, weights, _, _, _, logits = s.views
    blocks.route_experts(*s.views, renormalize=c["renormalize"])
    result = {"weights": s.weights, "experts": s.chosen, "offsets": s.offsets, "tokens": s.order, "slots": s.slots}
    if c["backward"]:
        blocks.route_experts_gradient(*s.gradient_views, weights, experts, logits, renormalize=c["renormalize"])
        result["logits_gradient"] = s.logits_gradient
    return result


def _work_route(c):
    n, e, k = c["tokens"], c["experts"], c["chosen"]
    values, others = n * e + n * k, 4 * (3 * n * k + e + 1)
    flops = 4 * n * e + n * e * k
    if c["backward"]:
        values, others = values + n * e + 2 * n * k + (0 if c["renormalize"] else n * e), others + 4 * n * k
    return values, others, flops


def _exact_route(s):
    c = s.case
    n, e, k = c["tokens"], c["experts"], c["chosen"]
    logits = s.logits.cpu().numpy().astype(np.float64)
    at = np.argsort(-logits, axis=1, kind="stable")[:, :k]
    values = np.take_along_axis(logits, at, 1)
    p = np.exp(logits - values[:, :1])
    if c["renormalize"]:
        inside = np.zeros((n, e), bool)
        np.put_along_axis(inside, at, True, 1)
        p = np.where(inside, p, 0.0)
    p /= p.sum(1, keepdims=True)
    weights = np.take_along_axis(p, at, 1)
    experts = np.where(np.isneginf(values), -1, at)
    flat = experts.reshape(-1)
    groups = [np.flatnonzero(flat == i) for i in range(e)]
    order = np.concatenate(groups)
    tokens, slots = np.full(n * k, -1), np.full(n * k, -1)
    tokens[:len(order)] = order // k
    slots[order] = np.arange(len(order))
    result = {"weights": weights, "experts": experts.astype(np.int32),
              "offsets": np.cumsum([0] + [len(g) for g in groups]).astype(np.int32), "tokens": tokens.astype(np.int32),
              "slots": slots.reshape(n, k).astype(np.int32)}
    if c["backward"]:
        dw = np.zeros((n, e))
        np.put_along_axis(dw, at, s.weights_gradient.cpu().numpy().astype(np.float64), 1)
        result["logits_gradient"] = p * (dw - (p * dw).sum(1, keepdims=True))
    return result


# ------------------------------------------------------------------------------------------------- products by expert

def _groups(s, assignments):
    """How many rows each expert has: uneven by the case's skew."""
    e = s.case["experts"]
    liked = np.exp(s.host.normal(0.0, s.case.get("skew", 0.5), e))
    return s.host.multinomial(assignments, liked / liked.sum())


def _prepare_products(s):
    c = s.case
    n, k, e, n_in, n_out = c["tokens"], c["chosen"], c["experts"], c["inputs"], c["outputs"]
    sizes = _groups(s, n * k)
    s.sizes, s.most = sizes, int(sizes.max())
    offsets = np.concatenate([[0], np.cumsum(sizes)])
    s.offsets = s.indexes(offsets)
    order = s.host.permutation(n * k) // k
    s.tokens = s.indexes(order)
    s.input, s.weights = s.normal(n, n_in), s.normal(e, n_out, n_in, std=1.0 / math.sqrt(n_in))
    s.result = s.empty(n * k, n_out)
    if c["backward"]:
        s.result_gradient = s.normal(n * k, n_out, std=1e-2)
        s.rows_gradient, s.weights_gradient = s.empty(n * k, n_in), s.empty(e, n_out, n_in)


def _plain_products(s):
    # the groups side by side, each as long as the longest
    c = s.case
    rows, e = c["tokens"] * c["chosen"], c["experts"]
    row = torch.arange(rows, device="cuda")
    group = torch.searchsorted(s.offsets[1:].contiguous(), row.to(torch.int32), right=True)
    place = row - s.offsets[group]
    spread = lambda t: t.new_zeros(e, s.most, t.shape[1]).index_put((group, place), t)
    taken = spread(s.input[s.tokens.long()])
    result = {"result": torch.bmm(taken, s.weights.transpose(1, 2).contiguous())[group, place]}
    if c["backward"]:
        gradient = spread(s.result_gradient)
        result["rows_gradient"] = torch.bmm(gradient, s.weights)[group, place]
        result["weights_gradient"] = torch.bmm(gradient.transpose(1, 2).contiguous(), taken)
    return result


def _own_products(s):
    from cortex_amd import blocks
    c = s.case
    if not hasattr(s, "views"):
        s.views = [s.view(t) for t in (s.result, s.input, s.weights, s.offsets, s.tokens)]
        if c["backward"]:
            s.gradient_views = [s.view(t) for t in (s.result_gradient, s.rows_gradient, s.weights_gradient)]
    result, input, weights, offsets, tokens = s.views
    blocks.grouped_gemm(result, True, 1.0, input, weights, 0.0, offsets, index=tokens)
    if not c["backward"]:
        return {"result": s.result}
    result_gradient, rows_gradient, weights_gradient = s.gradient_views
    blocks.grouped_gemm(rows_gradient, False, 1.0, result_gradient, weights, 0.0, offsets)
    blocks.grouped_gemm_weights(weights_gradient, 1.0, result_gradient, input, 0.0, offsets, b_index=tokens)
    return {"result": s.result, "rows_gradient": s.rows_gradient, "weights_gradient": s.weights_gradient}


def _work_products(c):
    n, k, e, n_in, n_out = c["tokens"], c["chosen"], c["experts"], c["inputs"], c["outputs"]
    rows = n * k
    weights = min(e, rows) * n_in * n_out
    values, flops = n * n_in + rows * n_out + weights, 2 * rows * n_in * n_out
    if c["backward"]:
        values, flops = values + rows * n_out + rows * n_in + e * n_in * n_out, 3 * flops
    return values, 4 * (rows + e), flops


def _exact_products(s):
    c = s.case
    rows, weights = s.input.double()[s.tokens.long()], s.weights.double()
    gradient = s.result_gradient.double() if c["backward"] else None
    result, rows_gradient, weights_gradient, at = [], [], [], 0
    for i, size in enumerate(s.sizes.tolist()):
        part = rows[at:at + size]
        result.append(part @ weights[i].t())
        if c["backward"]:
            rows_gradient.append(gradient[at:at + size] @ weights[i])
            weights_gradient.append(gradient[at:at + size].t() @ part)
        at += size
    found = {"result": torch.cat(result)}
    if c["backward"]:
        found.update(rows_gradient=torch.cat(rows_gradient), weights_gradient=torch.stack(weights_gradient))
    return found


# ------------------------------------------------------------------------------------------------- a token's results

def _prepare_combine(s):
    c = s.case
    n, k, d = c["tokens"], c["chosen"], c["width"]
    # which of the rows are a token's: in order of experts, tokens in their order within one; some have no row
    experts = s.host.integers(0, c["experts"], (n, k))
    dropped = s.host.permutation(n * k).reshape(n, k) < int(c["dropped"] * n * k)
    flat = np.where(dropped, c["experts"], experts).reshape(-1)
    order = np.argsort(flat, kind="stable")
    slots = np.empty(n * k, np.int64)
    slots[order] = np.arange(n * k)
    s.slots = s.indexes(np.where(dropped.reshape(-1), -1, slots).reshape(n, k))
    s.kept = int(n * k - dropped.sum())
    # a program keeps room for all the rows; the last ones are no token's when some were dropped
    s.rows = s.normal(n * k, d)
    weights = s.normal(n, k).exp()
    s.weights = weights / weights.sum(1, keepdim=True)
    s.output = s.empty(n, d)
    if c["backward"]:
        s.output_gradient = s.normal(n, d, std=1e-2)
        s.rows_gradient, s.weights_gradient = s.empty(n * k, d), s.empty(n, k)


def _plain_combine(s):
    c = s.case
    n, k, d = c["tokens"], c["chosen"], c["width"]
    have = s.slots >= 0
    at = s.slots.clamp(min=0).long()
    weights = torch.where(have, s.weights, 0.0)
    taken = s.rows[at]
    result = {"output": (weights[:, :, None] * taken).sum(1)}
    if c["backward"]:
        result["weights_gradient"] = torch.where(have, (taken * s.output_gradient[:, None, :]).sum(2), 0.0)
        spread = (weights[:, :, None] * s.output_gradient[:, None, :]).reshape(n * k, d)
        # rows of no token come after all others
        places = torch.where(have.reshape(-1), s.slots.reshape(-1).long(), n * k)
        result["rows_gradient"] = spread.new_empty(n * k + 1, d).index_copy(0, places, spread)[:s.kept]
    return result


def _own_combine(s):
    from cortex_amd import blocks
    c = s.case
    if not hasattr(s, "views"):
        s.views = [s.view(t) for t in (s.output, s.rows, s.weights, s.slots)]
        if c["backward"]:
            s.gradient_views = [s.view(t) for t in (s.rows_gradient, s.weights_gradient, s.output_gradient)]
    output, rows, weights, slots = s.views
    blocks.combine_experts(output, rows, weights, slots)
    if not c["backward"]:
        return {"output": s.output}
    blocks.combine_experts_gradient(*s.gradient_views, rows, weights, slots)
    return {"output": s.output, "weights_gradient": s.weights_gradient, "rows_gradient": s.rows_gradient[:s.kept]}


def _work_combine(c):
    n, k, d = c["tokens"], c["chosen"], c["width"]
    values, flops = n * k * d + n * d + n * k, 2 * n * k * d
    if c["backward"]:
        values, flops = values + n * d + 2 * n * k * d + 2 * n * k, flops + 3 * n * k * d
    return values, 4 * n * k * (2 if c["backward"] else 1), flops


def _exact_combine(s):
    c = s.case
    slots, weights, rows = s.slots.cpu().numpy(), s.weights.double(), s.rows.double()
    output = torch.zeros_like(s.output, dtype=torch.float64)
    found = {"output": output}
    if c["backward"]:
        gradient = s.output_gradient.double()
        found["weights_gradient"] = torch.zeros_like(weights)
        found["rows_gradient"] = torch.zeros_like(rows)
    for j in range(c["chosen"]):
        token = np.flatnonzero(slots[:, j] >= 0)
        row, token = torch.from_numpy(slots[token, j].astype(np.int64)).cuda(), torch.from_numpy(token).cuda()
        output[token] += weights[token, j, None] * rows[row]
        if c["backward"]:
            found["weights_gradient"][token, j] = (gradient[token] * rows[row]).sum(1)
            found["rows_gradient"][row] = weights[token, j, None] * gradient[token]
    if c["backward"]:
        found["rows_gradient"] = found["rows_gradient"][:s.kept]
    return found


# ------------------------------------------------------------------------------------------------- the norm of all gradients

def _clip_sizes(c):
    """Sizes spread as a network's are, the same for every seed: matrices, and many small vectors between them."""
    shares = np.random.default_rng(c["tensors"]).lognormal(0.0, 2.0, c["tensors"])
    return np.clip((shares / shares.sum() * c["values"]).astype(np.int64), 1, c["most"]).tolist()


def _prepare_clip(s):
    s.sizes = _clip_sizes(s.case)
    s.gradients = [s.normal(size, std=10.0 ** s.host.uniform(-3, -1)) for size in s.sizes]
    s.clipped = s.empty(sum(s.sizes))
    s.norm = s.empty(2)


def _plain_clip(s):
    squares = torch.stack([(g * g).sum() for g in s.gradients])
    norm = squares.sum().sqrt()
    factor = s.case["limit"] / torch.clamp(norm, min=s.case["limit"])
    return {"clipped": torch.cat(s.gradients) * factor, "norm": torch.stack([norm, factor])}


def _own_clip(s):
    from cortex_amd import optimize, tensor
    if not hasattr(s, "views"):
        s.views = [s.view(g) for g in s.gradients]
        # side by side in one buffer, as the state of an optimizer is
        flat, ends = s.view(s.clipped).buffer, np.cumsum(s.sizes).tolist()
        s.into = [flat.sub_buffer(end - size, size) for end, size in zip(ends, s.sizes)]
        s.norm_view = s.view(s.norm)
        s.backend = optimize.Backend(tensor.check_stream(), s.case["datatype"])
    optimize.clip_gradients(s.backend, s.views, s.case["limit"], s.norm_view, s.into)
    return {"clipped": s.clipped, "norm": s.norm}


def _work_clip(c):
    values = sum(_clip_sizes(c))
    return 2 * values + 2, 0, 3 * values


def _exact_clip(s):
    total = math.fsum(float((g.double() ** 2).sum()) for g in s.gradients)
    norm = math.sqrt(total)
    factor = min(1.0, s.case["limit"] / norm)
    return {"clipped": torch.cat([g.double() * factor for g in s.gradients]),
            "norm": torch.tensor([norm, factor], dtype=torch.float64)}


_PREPARE = {"norm": _prepare_norm, "route": _prepare_route, "products": _prepare_products, "combine": _prepare_combine,
            "clip": _prepare_clip}
_PLAIN = {"norm": _plain_norm, "route": _plain_route, "products": _plain_products, "combine": _plain_combine,
          "clip": _plain_clip}
_OWN = {"norm": _own_norm, "route": _own_route, "products": _own_products, "combine": _own_combine, "clip": _own_clip}
_WORK = {"norm": _work_norm, "route": _work_route, "products": _work_products, "combine": _work_combine, "clip": _work_clip}
_EXACT = {"norm": _exact_norm, "route": _exact_route, "products": _exact_products, "combine": _exact_combine,
          "clip": _exact_clip}
