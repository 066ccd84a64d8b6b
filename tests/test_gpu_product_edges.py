"""Products whose only terms lie at an edge: in the last, partial step of a contraction, on either side of a step's or a tile's border,
in the last rows or columns. A step, a row or a column that is lost is then the whole result, not a small part of it. And how
far results of random operands are off as a whole, which element-wise bounds that grow with the depth do not hold."""

import math

import pytest
import torch

from jax_linear_attention_b200 import layers

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def _edges(n, step):
    """Index sets of a range of n: its ends, the last partial step, both sides of borders of steps."""
    last = (n - 1) // step * step
    some = [[0], [n - 1], list(range(last, n))]
    for border in {step, 128, 256, 512, last, 16384}:
        if 0 < border < n:
            some.append([border - 1, border])
    return some


def _close(got, want, terms, dtype):
    """`terms` products an element, added in float32 (2^-23 of their sizes' sum each) and rounded: half a step."""
    size = want[1] if isinstance(want, tuple) else want.abs()
    want = want[0] if isinstance(want, tuple) else want
    off = (got.double() - want).abs() - torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2.0 ** -7) - terms * 2.0 ** -22 * size - 2.0 ** -24
    assert float(off.max()) <= 0, float(off.max())


def _product(a, b):
    """(a @ b, |a| @ |b|) in 64 bits."""
    a, b = a.double(), b.double()
    return a @ b, a.abs() @ b.abs()


# (rows, in, out): few tokens, pairs with one tile width and the other, tiles in halves and whole, several a pair
SIZES = [(5, 2048, 136), (50, 1000, 72), (100, 328, 264), (300, 72, 56), (1003, 520, 328), (8300, 72, 56), (8300, 264, 200),
         (18900, 72, 256), (33000, 136, 72)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, depth, out", SIZES)
def test_edges_of_the_contractions(rows, depth, out, dtype):
    dtype = DTYPES[dtype]
    x, w, dy = (_randn(k, *s).to(dtype) for k, s in ((1, (rows, depth)), (2, (out, depth)), (3, (rows, out))))

    def only(t, index, dim):
        kept = torch.zeros_like(t)
        kept.index_copy_(dim, index, t.index_select(dim, index))
        return kept

    for at in _edges(depth, 64):  # forward: over the inputs
        i = torch.tensor(at, device="cuda")
        _close(layers.linear(only(x, i, 1), w), _product(x[:, i], w[:, i].t()), len(at), dtype)
        up = only(w, i, 1)
        g, u = x[:, i].double() @ w[:, i].double().t(), x[:, i].double() @ w[:, i].double().t()
        h = layers.gated_linear(x, up, up, activation="sigmoid")
        want = torch.sigmoid(g) * u
        # float32 sums and activation: 2^-20 of what they are made of
        size = _product(x[:, i], w[:, i].t())[1]
        assert bool(((h.double() - want).abs() <= torch.finfo(dtype).eps / 2 * 1.01 * want.abs() + 2.0 ** -20 * (1 + size) ** 2).all())
    for at in _edges(rows, 64):  # dW: over the tokens
        i = torch.tensor(at, device="cuda")
        a, leaf = only(x, i, 0), w.clone().requires_grad_()
        dw, = torch.autograd.grad(layers.linear(a, leaf), [leaf], dy)
        _close(dw, _product(dy[i].t(), x[i]), len(at), dtype)
        dw, = torch.autograd.grad(layers.linear(x, leaf), [leaf], only(dy, i, 0))
        _close(dw, _product(dy[i].t(), x[i]), len(at), dtype)
        leaf_x = x.clone().requires_grad_()  # and dx, row by row: nothing but those rows
        dx, = torch.autograd.grad(layers.linear(leaf_x, w), [leaf_x], only(dy, i, 0))
        _close(dx[i], _product(dy[i], w), out, dtype)
        dx[i] = 0
        assert not bool(dx.any())
    for at in _edges(out, 64):  # dx: over the outputs
        i = torch.tensor(at, device="cuda")
        leaf = x.clone().requires_grad_()
        dx, = torch.autograd.grad(layers.linear(leaf, w), [leaf], only(dy, i, 1))
        _close(dx, _product(dy[:, i], w[i]), len(at), dtype)


def _rms(t):
    return float(t.double().square().mean().sqrt())


def _spread(a, b, half):
    """The root mean square that errors of up to `half` of a's elements, independent and to either side, leave in a @ b: half / sqrt(3)
    (an even spread) of the root of the products' squares' sum; three times that is the bound."""
    return 3 * half / math.sqrt(3) * float((a.double().square() @ b.double().square()).mean().sqrt())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, depth, out", SIZES + [(8300, 136, 1000), (2100, 520, 1000)])
def test_how_far_off_as_a_whole(rows, depth, out, dtype):
    dtype = DTYPES[dtype]
    half = torch.finfo(dtype).eps / 2
    x, w, up, dy = ((_randn(k, *s) * f).to(dtype) for k, s, f in ((1, (rows, depth), 1), (2, (out, depth), depth ** -0.5),
                                                                  (3, (out, depth), depth ** -0.5), (4, (rows, out), 1)))
    leaves = [t.requires_grad_() for t in (x, w, up)]
    wide = [t.detach().double().requires_grad_() for t in leaves]
    g, u = wide[0] @ wide[1].t(), wide[0] @ wide[2].t()
    h64 = torch.nn.functional.silu(g) * u
    dg, du = torch.autograd.grad(h64, [g, u], dy.double(), retain_graph=True)
    want = [h64.detach(), *torch.autograd.grad(h64, wide, dy.double())]
    h = layers.gated_linear(*leaves)
    got = [h, *torch.autograd.grad(h, leaves, dy)]
    x64, w64, up64 = (t.detach() for t in wide)
    # rounded results: half a step at most; dg and du rounded on the way to the products; float32 sums, activations and
    # TINY (float16 below its normal numbers) far below both
    through = [0, _spread(dg, w64, half) + _spread(du, up64, half), _spread(dg.t(), x64, half), _spread(du.t(), x64, half)]
    for a, b, t in zip(got, want, through):
        assert _rms(a.detach().double() - b) <= (half + 2.0 ** -15) * _rms(b) + t + 2.0 ** -24
    y = layers.linear(x, w)
    got = torch.autograd.grad(y, [x, w], dy)
    want = [x64 @ w64.t(), dy.double() @ w64, dy.double().t() @ x64]
    for a, b in zip([y, *got], want):
        assert _rms(a.detach().double() - b) <= (half + 2.0 ** -15) * _rms(b) + 2.0 ** -24


@pytest.mark.parametrize("rows", [12, 400, 8300])
def test_gradients_against_differences_a_row_at_a_time(rows):
    """Directions within one row (of x), or within one row of a weight: the slope is a row's own, and nothing else hides in it."""
    dtype = torch.float16
    x, w, up, dy = ((_randn(k, *s) * f).to(dtype) for k, s, f in ((1, (rows, 64), 1), (2, (72, 64), 0.125), (3, (72, 64), 0.125),
                                                                  (4, (rows, 72), 1)))
    leaves = [t.requires_grad_() for t in (x, w, up)]
    got = torch.autograd.grad(layers.gated_linear(*leaves), leaves, dy)
    wide = [t.detach().double() for t in leaves]

    def loss(args):
        return float((torch.nn.functional.silu(args[0] @ args[1].t()) * (args[0] @ args[2].t()) * dy.double()).sum())

    h, half = 2.0 ** -14, 2.0 ** -11
    g, u = wide[0] @ wide[1].t(), wide[0] @ wide[2].t()
    s = torch.sigmoid(g)
    dg, du = dy.double() * u * s * (1 + g * (1 - s)), dy.double() * g * s
    for k in range(3):
        n = wide[k].shape[0]
        for row in {0, 1, n // 2, n - 1, *(r for r in (31, 32, 63, 64, 127, 128, 255, 256, 511, 8191) if r < n)}:
            d = torch.zeros_like(wide[k])
            d[row] = _randn(row, 64).double()
            up_, down = (loss([v + (f * h * d if j == k else 0) for j, v in enumerate(wide)]) for f in (1, -1))
            slope, mine = (up_ - down) / (2 * h), float((got[k].double() * d).sum())
            # the gradient's rounding, and that of dg and du on their way to it: independent, so that their squares add up;
            # three times the root of the sum of squares (every one of them at its largest)
            if k == 0:
                inner = torch.cat([dg[row][:, None] * wide[1] * d[row], du[row][:, None] * wide[2] * d[row]])
            else:
                inner = (dg if k == 1 else du)[:, row][:, None] * wide[0] * d[row]
            # (a dg's rounding is the same for all columns of the direction: its terms add up first)
            off = 3 * half * math.sqrt(float((got[k][row].double() * d[row]).square().sum()) + float(inner.sum(1).square().sum()))
            assert abs(slope - mine) <= off + 2.0 ** -20 * (1 + abs(slope)) + 2.0 ** -16 * float(inner.abs().sum()) * h
