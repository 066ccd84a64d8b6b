"""Long contractions of the products: one sum over all tokens of a training step (the gradient of a weight), over very wide inputs
or outputs. The tensor cores cut every addition off instead of rounding it, so the error of one long sum grows with its
length, to one side. Here all terms are positive, the case in which it shows: no result may be further off than a sum in parts of
1024 additions each, joined with rounding, explains.

The bounds. An instruction adds 16 products (32 in e4m3) to the sum so far and cuts the result off to float32's 24 bits: at most
2^-23 of it. 1024 of them in a part: at most 2^-13 of the part's sum, all to the same side. The parts, up to 400 of them here, are joined
with rounding, 2^-24 each: another 2^-15 at most. e4m3's instructions may keep fewer bits of a term, 2^-13 of the largest. So PART
= 2^-13 + 2^-15 of a sum of positive terms (e4m3: 2^-13 more)."""

import pytest
import torch

from jax_linear_attention_b200 import _lib, layers

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": (torch.bfloat16, 0), "f16": (torch.float16, 1)}
PART = 2.0 ** -13 + 2.0 ** -15


def _positive(seed, *shape, dtype=torch.bfloat16, size=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (size * (0.5 + torch.rand(*shape, generator=gen, device="cuda"))).to(dtype)


def _product(a, b):
    """a.t() @ b in 64 bits, a part of the rows at a time."""
    return sum(a[i:i + 65536].double().t() @ b[i:i + 65536].double() for i in range(0, a.shape[0], 65536))


def _check_f32(got, want, part=PART):
    off = ((got.double() - want) / want).abs()
    assert float(off.max()) <= part, float(off.max())


def _check_rounded(got, want, dtype):
    """Rounding keeps the order of values: a sum between (1 - PART) and (1 + PART) of the exact one is rounded to something between
    their roundings. (The limits a little further apart: 64 bits are rounded to 32 on their way.)"""
    part = PART + 2.0 ** -22
    low, high = (want * (1 - part)).to(dtype), (want * (1 + part)).to(dtype)
    assert bool(((got >= low) & (got <= high)).all()), float(((got.double() - want) / want).abs().max())


def _weight_gradient(dz, x, dz2=None):
    rows, out = dz.shape
    dw = [torch.empty(out, x.shape[1], dtype=x.dtype, device="cuda") for _ in range(1 if dz2 is None else 2)]
    _lib.launch("jla_linear_bwd_weight", dz.device, 0 if x.dtype == torch.bfloat16 else 1, rows, x.shape[1], out, dz.data_ptr(),
                None if dz2 is None else dz2.data_ptr(), x.data_ptr(), x.stride(0), dw[0].data_ptr(),
                None if dz2 is None else dw[1].data_ptr())
    return dw


# rows of up to 128 and of more features (two tile widths), tiles in halves and whole, several tiles a pair of CTAs; more rows
# than 16384 by one step, by a part of one, by many times
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, depth, out", [(16384, 64, 72), (16385, 64, 72), (16448, 264, 200), (33000, 520, 72),
                                              (400_003, 64, 64), (400_003, 136, 264), (1_100_000, 64, 64), (40_000, 1792, 2560)])
def test_weight_gradient_of_many_tokens(rows, depth, out, dtype):
    dtype = DTYPES[dtype][0]
    size = min(1.0, (20000 / rows) ** 0.5)  # (sums that float16 holds)
    dz, x = _positive(1, rows, out, dtype=dtype, size=size), _positive(2, rows, depth, dtype=dtype, size=size)
    dw, = _weight_gradient(dz, x)
    _check_rounded(dw, _product(dz, x), dtype)


@pytest.mark.parametrize("rows, depth, out", [(50_001, 72, 136), (131_072, 264, 264), (20_000, 2048, 2048)])
def test_both_weight_gradients_of_many_tokens(rows, depth, out):
    size = min(1.0, (20000 / rows) ** 0.5)
    dz, dz2, x = (_positive(s, rows, n, dtype=torch.float16, size=size) for s, n in ((1, out), (2, out), (3, depth)))
    for got, d in zip(_weight_gradient(dz, x, dz2), (dz, dz2)):
        _check_rounded(got, _product(d, x), torch.float16)


def test_weight_gradient_through_the_layer():
    rows = 300_000
    x = _positive(1, rows, 64, size=0.25).requires_grad_()
    w = _positive(2, 72, 64, size=0.1).requires_grad_()
    dy = _positive(3, rows, 72, size=0.25)
    dx, dw = torch.autograd.grad(layers.linear(x, w), [x, w], dy)
    _check_rounded(dw, _product(dy, x.detach()), torch.bfloat16)
    _check_rounded(dx, dy.double() @ w.detach().double(), torch.bfloat16)


@pytest.mark.parametrize("rows, depth, out", [(1, 131_072, 72), (20, 262_136, 136), (100, 262_136, 264), (600, 70_000, 72),
                                              (300, 262_136, 264), (4, 40_000, 20_000), (2100, 33_000, 2600)])
def test_product_of_very_wide_inputs(rows, depth, out):
    for dtype, code in DTYPES.values():
        x, w = _positive(1, rows, depth, dtype=dtype), _positive(2, out, depth, dtype=dtype, size=2.0 ** -5)
        y, z = torch.empty(rows, out, dtype=dtype, device="cuda"), torch.empty(rows, out, device="cuda")
        _lib.launch("jla_linear_fwd", x.device, code, code, rows, depth, out, x.data_ptr(), depth, w.data_ptr(), None, None, None, 0,
                    None, y.data_ptr(), z.data_ptr())
        want = _product(x.t(), w.t())
        _check_f32(z, want)
        assert bool((y == z.to(dtype)).all())


@pytest.mark.parametrize("rows, depth, out", [(3, 100_000, 72), (50, 262_136, 136), (300, 70_000, 72), (300, 70_000, 328),
                                              (9400, 20_000, 136)])
def test_gated_product_of_very_wide_inputs(rows, depth, out):
    x = _positive(1, rows, depth)
    w, up = (_positive(s, out, depth, size=1 / depth) for s in (2, 3))
    h = torch.empty(rows, out, dtype=torch.bfloat16, device="cuda")
    g, u = (torch.empty(rows, out, device="cuda") for _ in range(2))
    _lib.launch("jla_gated_linear_fwd", x.device, 0, 0, rows, depth, out, x.data_ptr(), depth, w.data_ptr(), up.data_ptr(), None, None,
                None, 3, h.data_ptr(), g.data_ptr(), u.data_ptr())
    _check_f32(g, _product(x.t(), w.t()))
    _check_f32(u, _product(x.t(), up.t()))
    want = torch.sigmoid(g.double()) * u.double()
    assert bool(((h.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -18) * want).all())


@pytest.mark.parametrize("rows, depth, out", [(5, 300_000, 72), (100, 300_000, 264), (600, 100_000, 72), (300, 300_000, 264)])
def test_input_gradient_of_very_wide_outputs(rows, depth, out):
    """(depth: the outputs that are summed over)"""
    for pair in (False, True):
        dz, dz2 = (_positive(s, rows, depth, dtype=torch.float16, size=0.25) for s in (1, 2))
        w, w2 = (_positive(s, depth, out, dtype=torch.float16, size=0.125) for s in (3, 4))
        dx = torch.empty(rows, out, dtype=torch.float16, device="cuda")
        _lib.launch("jla_linear_bwd_input", dz.device, 1, rows, out, depth, dz.data_ptr(), w.data_ptr(),
                    dz2.data_ptr() if pair else None, w2.data_ptr() if pair else None, dx.data_ptr())
        want = _product(dz.t(), w) + (_product(dz2.t(), w2) if pair else 0)
        _check_rounded(dx, want, torch.float16)


@pytest.mark.parametrize("rows, depth, out", [(2, 262_144, 72), (40, 524_288, 136), (300, 524_288, 264), (600, 100_000, 72)])
def test_e4m3_products_of_very_wide_inputs(rows, depth, out):
    x, w, up = (_positive(s, n, depth, dtype=torch.float8_e4m3fn, size=8) for s, n in ((1, rows), (2, out), (3, out)))
    xs, ws, us = (_positive(s, n, dtype=torch.float32) for s, n in ((4, rows), (5, out), (6, out)))
    y, h = (torch.empty(rows, out, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    z, g, u = (torch.empty(rows, out, device="cuda") for _ in range(3))
    _lib.launch("jla_linear_fwd", x.device, 3, 0, rows, depth, out, x.data_ptr(), depth, w.data_ptr(), xs.data_ptr(), ws.data_ptr(),
                None, 0, None, y.data_ptr(), z.data_ptr())
    _lib.launch("jla_gated_linear_fwd", x.device, 3, 0, rows, depth, out, x.data_ptr(), depth, w.data_ptr(), up.data_ptr(),
                xs.data_ptr(), ws.data_ptr(), us.data_ptr(), 3, h.data_ptr(), g.data_ptr(), u.data_ptr())
    for got, m, s in ((z, w, ws), (g, w, ws), (u, up, us)):
        _check_f32(got, _product(x.float().t(), m.float().t()) * xs.double()[:, None] * s.double(), PART + 2.0 ** -13)


def test_long_sums_give_the_same_bits():
    dz, x = (torch.randn(70_000, n, device="cuda").bfloat16() for n in (200, 264))
    first, = _weight_gradient(dz, x)
    for _ in range(3):
        assert bool((_weight_gradient(dz, x)[0] == first).all())


def test_infinities_and_nan_of_one_part_reach_the_sum():
    dz, x = (torch.randn(60_000, n, device="cuda").bfloat16() for n in (64, 136))
    clean, = _weight_gradient(dz, x)
    for row in (3, 30_000, 59_999):
        bad = x.clone()
        bad[row, 7] = float("nan")
        dw, = _weight_gradient(dz, bad)
        keep = [i for i in range(136) if i != 7]
        assert bool(dw[:, 7].isnan().all()) and bool((dw[:, keep] == clean[:, keep]).all())
