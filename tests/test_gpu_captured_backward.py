"""Backward passes that are captured into a graph: a leaf whose gradient would be handed over outside of the capture is found
wherever it stands, also behind torch's own nodes, and nothing else is refused."""

import pytest
import torch

from jax_linear_attention_b200 import layers

pytestmark = pytest.mark.gpu


def _leaf(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda").to(dtype).requires_grad_()


def _cases():
    x, w, wide, odd, b = _leaf(64, 64), _leaf(64, 64), _leaf(64, 160), _leaf(63, 60), _leaf(64)
    n = _leaf(64)
    d, e = x.detach(), w.detach()
    return {"bias": (lambda: layers.linear(d, e, b), b), "transposed": (lambda: layers.linear(d, w.t()), w),
            "padded": (lambda: layers.linear(d[:, :60], odd), odd), "slice": (lambda: layers.linear(wide[:, 8:72], e), wide),
            "gate": (lambda: layers.gated_linear(d, w.t(), e), w), "up": (lambda: layers.gated_linear(d, e, 2 * w), w),
            "norm": (lambda: layers.rms_norm(d, n), n), "two": (lambda: layers.linear(layers.linear(x, e), e), x),
            "far": (lambda: layers.linear((x.float() * 2 + 1).bfloat16().view(32, 128).view(64, 64), e), x)}


def _step(call, leaf):
    y = call()
    return torch.autograd.grad(y, [leaf], torch.ones_like(y))[0]


@pytest.mark.parametrize("name", ["bias", "transposed", "padded", "slice", "gate", "up", "norm", "two", "far"])
def test_leaf_behind_other_nodes(name):
    call, leaf = _cases()[name]
    want = _step(call, leaf)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(call, leaf)
    torch.cuda.synchronize()
    alive = call()
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            _step(call, leaf)
    del alive
    alive = _leaf(4, 4) * 2  # of another leaf
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(call, leaf)
    graph.replay()
    assert bool((out == want).all())
    del alive


def test_part_of_the_graph_made_before_the_capture():
    x, w = _leaf(64, 64).detach(), _leaf(64, 64)
    wt = w.t()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = layers.linear(x, wt)
        torch.autograd.grad(y, [w], torch.ones_like(y), retain_graph=True)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="made there"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            y = layers.linear(x, wt)
            torch.autograd.grad(y, [w], torch.ones_like(y))


def test_other_leaves_of_the_same_graph_do_not_count():
    """A gradient that is not asked for is not handed over."""
    x, w = _leaf(64, 64), _leaf(64, 64)
    want = _step(lambda: layers.linear(x, w.t(), activation="silu"), x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(lambda: layers.linear(x, w.t(), activation="silu"), x)
    torch.cuda.synchronize()
    alive = w + 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(lambda: layers.linear(x, w.t(), activation="silu"), x)
    graph.replay()
    assert bool((out == want).all())
    del alive
