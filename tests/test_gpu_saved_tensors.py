"""The norm and the products under saved-tensor hooks: what comes back for the backward pass may lie in memory in another way than
what was saved (offloading packs a slice), and is refused where it is another tensor altogether."""

import pytest
import torch

from jax_linear_attention_b200 import layers

pytestmark = pytest.mark.gpu

hooks = torch.autograd.graph.saved_tensors_hooks


def _transposed(t):
    """The same values, columns next to each other in memory."""
    return t.flatten(0, -2).t().contiguous().t().view(t.shape) if t.ndim > 1 else t.flip(0).contiguous().flip(0)


def _odd_address(t):
    """The same values, not on 16 bytes."""
    return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)


def _apart(t):
    """The same values, rows that lie apart (by no multiple of 16 bytes)."""
    return torch.empty(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)[..., :t.shape[-1]].copy_(t)


OFFLOADS = {"cpu": lambda: torch.autograd.graph.save_on_cpu(), "pinned": lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
            "transposed": lambda: hooks(lambda t: t.clone(), _transposed), "odd": lambda: hooks(lambda t: t.clone(), _odd_address),
            "apart": lambda: hooks(lambda t: t.clone(), _apart), "wider": lambda: hooks(lambda t: t.clone(), lambda t: torch.cat(
                [t, t], -1)[..., :t.shape[-1]])}


def _calls(rows, start):
    """``(call, leaves, gradient)`` of every operator, x a slice of columns that starts at ``start``."""
    gen = torch.Generator(device="cuda").manual_seed(rows + start)

    def normal(*shape, size=1.0):
        return (size * torch.randn(*shape, generator=gen, device="cuda")).bfloat16().requires_grad_()

    wide, w, up, r, s = normal(rows, 160), normal(72, 64, size=0.125), normal(72, 64, size=0.125), normal(rows, 72), normal(rows, 64)
    b, n = (torch.randn(k, generator=gen, device="cuda").requires_grad_() for k in (72, 64))
    dy, dx = normal(rows, 72).detach(), normal(rows, 64).detach()
    x = wide[:, start:start + 64]
    return [(lambda: layers.linear(x, w), [wide, w], dy),
            (lambda: layers.linear(x, w, b, activation="silu", residual=r), [wide, w, b, r], dy),
            (lambda: layers.gated_linear(x, w, up), [wide, w, up], dy),
            (lambda: layers.rms_norm(x, n), [wide, n], dx),
            (lambda: layers.rms_norm(x, n, residual=s)[0], [wide, s, n], dx)]


@pytest.mark.parametrize("rows", [24, 300, 8300])
@pytest.mark.parametrize("start", [0, 16, 3])
@pytest.mark.parametrize("how", OFFLOADS)
def test_gradients_under_hooks(how, start, rows):
    for call, leaves, dy in _calls(rows, start):
        want = torch.autograd.grad(call(), leaves, dy)
        with OFFLOADS[how]():
            y = call()
        got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        assert all(bool((a == b).all()) for a, b in zip(got, want))
        for k, leaf in enumerate(leaves):  # one at a time
            g, = torch.autograd.grad(y, [leaf], dy, retain_graph=True)
            assert bool((g == want[k]).all())


def test_other_tensors_from_a_hook_are_refused():
    for change in (lambda t: t.double(), lambda t: t[:-1], lambda t: t.cpu(), lambda t: t.flatten(), lambda t: t[None]):
        for call, leaves, dy in _calls(40, 0):
            with hooks(lambda t: t, lambda t: change(t) if t.ndim > 1 else t):
                y = call()
            with pytest.raises(ValueError, match="from its hook"):
                torch.autograd.grad(y, leaves, dy)


def test_checkpointed_slices():
    from torch.utils.checkpoint import checkpoint

    for call, leaves, dy in _calls(300, 16):
        want = torch.autograd.grad(call(), leaves, dy)
        y = checkpoint(call, use_reentrant=False)
        assert all(bool((a == b).all()) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))
