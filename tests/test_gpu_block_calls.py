"""Further ways to call the norm and the products: graphed callables, compiled functions, functional transforms, gradients and operands that lie
oddly in memory, nothing at all in odd widths."""

import pytest
import torch

from jax_linear_attention_b200 import layers

pytestmark = pytest.mark.gpu


def _normal(*shape, dtype=torch.bfloat16, size=1.0):
    return (size * torch.randn(*shape, device="cuda")).to(dtype)


class Block(torch.nn.Module):
    def __init__(self, width=64, inner=72, bias_dtype=torch.float32):
        super().__init__()
        self.norm = torch.nn.Parameter(torch.ones(width, device="cuda"))
        self.gate, self.up = (torch.nn.Parameter(_normal(inner, width, size=0.125)) for _ in range(2))
        self.down = torch.nn.Parameter(_normal(inner, width, size=0.125))
        self.bias = torch.nn.Parameter(_normal(width, dtype=bias_dtype))

    def forward(self, x):
        h = layers.gated_linear(layers.rms_norm(x, self.norm), self.gate, self.up)
        return layers.linear(h, self.down.t(), self.bias, residual=x, activation="silu")


@pytest.mark.parametrize("bias_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [8, 300])
def test_graphed_callables(rows, bias_dtype):
    torch.manual_seed(rows)
    block = Block(bias_dtype=bias_dtype)
    graphed = torch.cuda.make_graphed_callables(block, (_normal(rows, 64).requires_grad_(),))
    for _ in range(3):
        x, dy = _normal(rows, 64).requires_grad_(), _normal(rows, 64)
        leaves = [x, *block.parameters()]
        y = graphed(x)
        got = [y.detach().clone(), *(g.clone() for g in torch.autograd.grad(y, leaves, dy))]
        z = Block.forward(block, x)
        assert all(bool((a == b).all()) for a, b in zip(got, [z, *torch.autograd.grad(z, leaves, dy)]))


def test_gradients_that_lie_oddly():
    x, w, up, n = _normal(24, 64).requires_grad_(), _normal(72, 64).requires_grad_(), _normal(72, 64).requires_grad_(), torch.ones(64, device="cuda")
    for call, leaves, out in ((lambda: layers.linear(x, w, activation="silu"), [x, w], 72), (lambda: layers.gated_linear(x, w, up), [x, w, up], 72),
                              (lambda: layers.rms_norm(x, n), [x], 64), (lambda: layers.linear(x, w, torch.zeros(72, device="cuda")), [x, w], 72)):
        dy = _normal(24, out)
        want = torch.autograd.grad(call(), leaves, dy)
        odd = _normal(24, out + 3)
        odd[:, 1:out + 1] = dy
        for same in (dy.t().contiguous().t(), odd[:, 1:out + 1], torch.empty(24 * out + 1, device="cuda").bfloat16()[1:].view(24, out).copy_(dy)):
            assert all(bool((a == b).all()) for a, b in zip(torch.autograd.grad(call(), leaves, same), want))
        y = call()
        got = torch.autograd.grad(y.float(), leaves, dy.float())
        assert all(bool((a == b).all()) for a, b in zip(got, want))


def test_operands_that_lie_oddly():
    x = _normal(6, 64)
    w, r, b = _normal(72, 64), _normal(6, 72), torch.randn(72, device="cuda")
    want = layers.linear(x, w, b, residual=r)

    def negated(t):  # a lazily negated view: -(-t)
        return torch._neg_view(-t)

    for a in (negated(x), x.view(3, 2, 64).transpose(0, 1).contiguous().transpose(0, 1), x.t().contiguous().t(), x.view(6, 1, 64)):
        assert bool((layers.linear(a, w, b, residual=r.view(*a.shape[:-1], 72)).view(6, 72) == want).all())
    for a in (negated(w), w.t().contiguous().t(), torch.cat([w, w], 1)[:, :64]):
        assert bool((layers.linear(x, a, b, residual=r) == want).all())
        g = layers.gated_linear(x, a, a)
        assert bool((g == layers.gated_linear(x, w, w)).all())
    assert bool((layers.linear(x, w, negated(b), residual=negated(r)) == want).all())
    big = _normal(5, 7, 3, 80)
    part = big[1:4, ::2, 1:2, 8:72]  # rows that lie apart by different amounts
    assert bool((layers.linear(part, w) == layers.linear(part.contiguous(), w)).all())
    part = big[:, 2:3, 1:2, 8:72]  # by one amount, behind dimensions of one
    assert bool((layers.linear(part, w) == layers.linear(part.contiguous(), w)).all())
    overlap = torch.as_strided(big.view(-1), (20, 64), (8, 1))  # rows that overlap
    assert bool((layers.linear(overlap, w) == layers.linear(overlap.contiguous(), w)).all())
    assert bool((layers.linear(big[0, 0, 0, :64:1], w) == layers.linear(big[0, 0, 0, :64].clone(), w)).all())
    assert bool((layers.linear(_s := big.view(-1)[:128:2], w) == layers.linear(_s.contiguous(), w)).all())


@pytest.mark.parametrize("depth, out", [(64, 72), (7, 5), (60, 72), (64, 70)])
def test_no_rows_of_any_width(depth, out):
    w, up, b = _normal(out, depth).requires_grad_(), _normal(out, depth).requires_grad_(), torch.zeros(out, device="cuda").requires_grad_()
    for shape in ((0, depth), (3, 0, depth), (0, 4, depth)):
        x = _normal(*shape).requires_grad_()
        r = _normal(*shape[:-1], out).requires_grad_()
        y = layers.linear(x, w, b, activation="gelu", residual=r)
        assert y.shape == (*shape[:-1], out)
        for g, leaf in zip(torch.autograd.grad(y.sum(), [x, w, b, r]), (x, w, b, r)):
            assert g.shape == leaf.shape and not bool(g.any())
        h = layers.gated_linear(x, w, up)
        for g, leaf in zip(torch.autograd.grad(h.sum(), [x, w, up]), (x, w, up)):
            assert g.shape == leaf.shape and not bool(g.any())


def test_functional_transforms_raise():
    """No rule for them, and no crash."""
    x, w, n = _normal(8, 64), _normal(72, 64), torch.ones(64, device="cuda")
    for call in (lambda v: layers.linear(v, w), lambda v: layers.gated_linear(v, w, w), lambda v: layers.rms_norm(v, n)):
        for transform in (lambda f: torch.func.grad(lambda v: f(v).float().sum()), lambda f: torch.func.jacrev(f),
                          lambda f: torch.func.functionalize(f), lambda f: torch.func.vmap(f)):
            with pytest.raises(Exception):
                transform(call)(x)


def test_compiled_around():
    """A compiled function breaks its graph at these calls, and computes the same."""
    torch.manual_seed(0)
    block = Block()
    x = _normal(40, 64).requires_grad_()
    dy = _normal(40, 64)
    want = block(x)
    grads = torch.autograd.grad(want, [x, *block.parameters()], dy)
    compiled = torch.compile(lambda v: block(v) * 1, backend="aot_eager")
    y = compiled(x)
    got = torch.autograd.grad(y, [x, *block.parameters()], dy)
    assert bool((y == want).all()) and all(bool((a == b).all()) for a, b in zip(got, grads))


def test_operands_that_are_no_tensors():
    x, w, n = _normal(8, 64), _normal(72, 64), torch.ones(64, device="cuda")
    q, s, qs = x.to(torch.float8_e4m3fn), torch.ones(8, device="cuda"), torch.ones(72, device="cuda")
    qw = w.to(torch.float8_e4m3fn)
    for call, text in ((lambda: layers.linear(x, w, 0.5), "bias"), (lambda: layers.linear(x, w, residual=[1.0]), "residual"),
                       (lambda: layers.linear(q, qw, x_scale=1.0, weight_scale=qs), "x_scale"),
                       (lambda: layers.linear(q, qw, x_scale=s, weight_scale=1.0), "weight_scale"),
                       (lambda: layers.gated_linear(q, qw, qw, x_scale=s, gate_scale=qs, up_scale=2), "up_scale"),
                       (lambda: layers.rms_norm(x, n, residual=0), "residual"), (lambda: layers.rms_norm(x, 1.0), "weight"),
                       (lambda: layers.linear(x, None), "weight 0"), (lambda: layers.gated_linear(x, w, None), "weight 1"),
                       (lambda: layers.linear(x, w, out_dtype="bf16"), "out_dtype")):
        with pytest.raises(ValueError, match=text):
            call()
