"""The operators of a residual block of experts run together: a block's gradients against differences, and a few training
steps (norm, routing, grouped products, combining, clipping, Adam) that lower a loss."""
import numpy as np
import pytest

from cortex_amd import blocks
from cortex_amd import capi
from cortex_amd import driver as drv
from cortex_amd import optimize
from cortex_amd import tensor as ct

pytestmark = pytest.mark.gpu


@pytest.fixture()
def as_released():
    """Debug-sync mode off, as a user runs, and on again for the other tests."""
    capi.call("ct_set_device", 0)
    capi.call("ct_set_debug_sync", 0)
    yield
    capi.call("ct_set_debug_sync", 1)


def made(rng, tokens, width, hidden, experts, datatype, biases):
    shapes = {"router": ([experts, width], 1.0), "first": ([experts, hidden, width], width ** -0.5),
              "second": ([experts, width, hidden], hidden ** -0.5)}
    host = {k: rng.standard_normal(s) * scale for k, (s, scale) in shapes.items()}
    host.update({"post-scale": 1 + 0.1 * rng.standard_normal(width), "pre-scale": 1 + 0.1 * rng.standard_normal(width),
                 "gate": 0.5 + 0.1 * rng.standard_normal((1, width))})
    if biases:
        host.update({"post-bias": 0.1 * rng.standard_normal(width), "pre-bias": 0.1 * rng.standard_normal(width)})
    return host


def on_device(host, datatype):
    return {k: {"buffer": ct.to_tensor(v, datatype), "gradient": ct.new_tensor(list(v.shape), datatype=datatype)} for k, v in host.items()}


@pytest.mark.parametrize("kinds,renormalize", [(("rms", "rms"), True), (("layer", "layer"), False)])
def test_a_block_s_gradients_are_the_differences(kinds, renormalize):
    """In double: central differences of step 1e-5 along one direction through every parameter and input.  The choice of
    experts and the signs under the activation do not change over such a step for these inputs; bar 1e-6."""
    capi.call("ct_set_device", 0)
    capi.call("ct_set_debug_sync", 1)
    stream = drv.HipDriver().default_device().create_stream()
    rng = np.random.default_rng(3)
    tokens, width, hidden, experts, chosen = 13, 24, 40, 5, 2
    host = made(rng, tokens, width, hidden, experts, "double", kinds[0] == "layer")
    host["x"], host["residual"] = rng.standard_normal((tokens, width)), rng.standard_normal((tokens, width))
    direction = {k: rng.standard_normal(v.shape) for k, v in host.items()}
    to_output, to_normalized = rng.standard_normal((tokens, width)), rng.standard_normal((tokens, width))
    with ct.tensor_context(stream, "double"):
        block = blocks.ExpertBlock(tokens, width, hidden, experts, chosen,
                                   blocks.norm_descriptor(post=kinds[0], pre=kinds[1], residual_scale=0.8), renormalize=renormalize)
        output, normalized = ct.new_tensor([tokens, width]), ct.new_tensor([tokens, width])
        read = lambda t: ct.to_double_array(t).reshape(t.shape())

        def value(step):
            p = on_device({k: v + step * direction[k] for k, v in host.items()}, "double")
            x, residual = p.pop("x"), p.pop("residual")
            block.forward(p, x["buffer"], residual["buffer"], output, normalized)
            return (read(output) * to_output).sum() + (read(normalized) * to_normalized).sum(), p, x, residual

        high, low = value(1e-5)[0], value(-1e-5)[0]
        _, p, x, residual = value(0.0)
        block.backward(p, x["buffer"], output, x["gradient"], residual["gradient"], ct.to_tensor(to_output), ct.to_tensor(to_normalized))
        p.update(x=x, residual=residual)
        along = sum((read(p[k]["gradient"]) * direction[k]).sum() for k in p)
        assert abs(along - (high - low) / 2e-5) <= 1e-6 * max(1.0, abs(along))
        for k in p:     # each parameter by itself
            assert np.linalg.norm(read(p[k]["gradient"])) > 0, k
    stream.release()


def test_a_few_training_steps_lower_the_loss(as_released):
    """Mean squared distance from the results of another block of the same kind: forward, backward, clipping, Adam."""
    stream = drv.HipDriver().default_device().create_stream()
    rng = np.random.default_rng(4)
    tokens, width, hidden, experts, chosen = 256, 64, 96, 8, 2
    x_host = rng.standard_normal((tokens, width))
    with ct.tensor_context(stream, "float"):
        block = blocks.ExpertBlock(tokens, width, hidden, experts, chosen)
        x = ct.to_tensor(x_host)
        new = lambda: ct.new_tensor([tokens, width])
        target, output, normalized, x_gradient, residual_gradient, difference = (new() for _ in range(6))
        block.forward(on_device(made(rng, tokens, width, hidden, experts, "float", True), "float"), x, x, output, target)
        p = on_device(made(rng, tokens, width, hidden, experts, "float", True), "float")
        norm = ct.new_tensor([2])
        count = sum(v["buffer"].ecount() for v in p.values())
        memory = {"m": ct.new_tensor([count]), "v": ct.new_tensor([count])}
        optimizer = optimize.create_optimizer(optimize.Backend(stream), optimize.adam(alpha=3e-3))
        losses, norms = [], []
        for _ in range(30):
            block.forward(p, x, x, output, normalized)
            ct.binary_op(difference, 1.0, normalized, 1.0, target, "-")
            losses.append(float((ct.to_double_array(difference) ** 2).mean()))
            block.backward(p, x, output, x_gradient, residual_gradient, None, difference)
            optimize.clip_gradients(optimizer.backend, [v["gradient"] for v in p.values()], 5.0, norm)
            norms.append(ct.to_double_array(norm))
            optimizer = optimizer.batch_update()
            at = 0
            for v in p.values():
                optimizer.compute_parameters(memory, 1.0, at, v["gradient"], v["buffer"])
                at += v["buffer"].ecount()
        assert all(np.isfinite(losses)) and losses[-1] < 0.6 * losses[0], losses
        assert norms[0][0] > 5.0 and abs(norms[0][1] - 5.0 / norms[0][0]) < 1e-6
        # what Adam last saw is within the limit
        squares = sum((ct.to_double_array(v["gradient"]) ** 2).sum() for v in p.values())
        assert np.sqrt(squares) <= 5.0 * (1 + 1e-5)
    stream.release()
