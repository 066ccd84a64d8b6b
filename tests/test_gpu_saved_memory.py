"""What the products keep alive for a backward pass: the operands of the gradients that are wanted, and no others."""

import pytest
import torch

from jax_linear_attention_b200 import layers

pytestmark = pytest.mark.gpu

ROWS, DEPTH, OUT = 300, 64, 72
X, W, Z = ROWS * DEPTH, OUT * DEPTH, ROWS * OUT  # elements of x, of a weight, of what is kept before an activation


def _kept(call, leaves):
    """The sizes of the saved tensors; the gradients are those of a call in which everything is differentiated."""
    sizes = []

    def pack(t):
        sizes.append(t.numel())
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = call()
    got = torch.autograd.grad(y, leaves, torch.ones_like(y))
    return sorted(sizes), got


def _operands(differentiated):
    gen = torch.Generator(device="cuda").manual_seed(4)
    shapes = {"x": (ROWS, DEPTH), "w": (OUT, DEPTH), "up": (OUT, DEPTH), "r": (ROWS, OUT)}
    t = {n: (torch.randn(*s, generator=gen, device="cuda") / 8).bfloat16() for n, s in shapes.items()}
    t["b"] = torch.randn(OUT, generator=gen, device="cuda")
    for n in differentiated:
        t[n].requires_grad_()
    return t


@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("names, kept", [("x", [W]), ("w", [X]), ("xw", [X, W]), ("b", []), ("r", []), ("xb", [W]), ("wr", [X])])
def test_linear(names, kept, act):
    def call(t):
        return lambda: layers.linear(t["x"], t["w"], t["b"], activation=act, residual=t["r"])

    t, all_ = _operands(names), _operands("xwbr")
    sizes, got = _kept(call(t), [t[n] for n in names])
    _, want = _kept(call(all_), [all_[n] for n in names])
    assert sizes == sorted(kept + ([Z] if act and names != "r" else []))
    assert all(bool((a == b).all()) for a, b in zip(got, want))


@pytest.mark.parametrize("names, kept", [(("x",), [W, W]), (("w",), [X]), (("up",), [X]), (("w", "up"), [X]), (("x", "up"), [X, W, W])])
def test_gated_linear(names, kept):
    def call(t):
        return lambda: layers.gated_linear(t["x"], t["w"], t["up"])

    t, all_ = _operands(names), _operands(("x", "w", "up"))
    sizes, got = _kept(call(t), [t[n] for n in names])
    _, want = _kept(call(all_), [all_[n] for n in names])
    assert sizes == sorted(kept + [Z, Z])
    assert all(bool((a == b).all()) for a, b in zip(got, want))
