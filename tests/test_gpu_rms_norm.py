"""``layers.rms_norm`` against its definition in 64 bits: widths that fill vectors and that do not, one row to many, rows of
zeros, infinities and NaN, the e4m3 form, gradients against the formula's and against differences."""

import pytest
import torch

from jax_linear_attention_b200 import layers

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def _inputs(rows, dim, dtype, residual, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, dim, generator=gen, device="cuda").to(dtype)
    r = (3 * torch.randn(rows, dim, generator=gen, device="cuda")).to(dtype) if residual else None
    w = 1 + 0.3 * torch.randn(dim, generator=gen, device="cuda")
    dy = torch.randn(rows, dim, generator=gen, device="cuda").to(dtype)
    ds = torch.randn(rows, dim, generator=gen, device="cuda").to(dtype)
    return x, r, w, dy, ds


def _reference(x, r, w):
    t = x.double() if r is None else x.double() + r.double()
    return t, t / torch.sqrt(t.square().mean(-1, keepdim=True) + EPS) * w.double()


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _close(got, want, rel, extra=0.0):
    """|got - want| <= rel |want| + extra, element by element; `extra` may be a tensor."""
    err = (got.double() - want).abs() - rel * want.abs()
    assert bool((err <= extra).all()), float((err - extra).max())


# float32 arithmetic of one value: the sum of dim squares (pairwise over threads: under 64 roundings in a row of any width
# here), the mean, the root (2 roundings), two products: 72 roundings of 2^-24 cover it.
F32_WORK = 72 * 2.0 ** -24


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, dim", [(1, 1), (1, 2048), (3, 7), (5, 64), (150, 72), (33, 1000), (257, 1001), (9, 2048),
                                       (300, 4096), (2, 4097), (200, 8192), (5, 16384), (3, 16383), (1, 8)])
@pytest.mark.parametrize("residual", [False, True])
def test_forward(rows, dim, dtype, residual):
    dtype = DTYPES[dtype]
    x, r, w, _, _ = _inputs(rows, dim, dtype, residual)
    t, want = _reference(x, r, w)
    out = layers.rms_norm(x, w, residual=r, eps=EPS)
    y, stream = out if residual else (out, None)
    assert y.dtype == dtype and y.shape == x.shape
    _close(y, want, _half_step(dtype) + F32_WORK, 2.0 ** -24)  # (the last: float16 below its normal numbers)
    if residual:
        _close(stream, t, _half_step(dtype) + 2.0 ** -24, 2.0 ** -24)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, dim, residual", [(1, 64, True), (5, 7, False), (300, 2048, True), (150, 4096, False),
                                                 (17, 1001, True), (4, 16384, True), (1, 16, False)])
def test_e4m3(rows, dim, dtype, residual):
    dtype = DTYPES[dtype]
    x, r, w, _, _ = _inputs(rows, dim, dtype, residual)
    x[0] = 0
    if r is not None:
        r[0] = 0
    t, want = _reference(x, r, w)
    out = layers.rms_norm(x, w, residual=r, eps=EPS, out_dtype=torch.float8_e4m3fn)
    q, scale = out[:2]
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (rows,) and scale.dtype == torch.float32
    assert float(scale[0]) == 1.0 and not bool(q[0].float().any())
    top = want.abs().amax(-1)
    _close(scale[1:], (top / 448)[1:], F32_WORK + 2.0 ** -24)
    # e4m3: half a step of 2^-3, or of the subnormal numbers' step of 2^-9
    _close(q.double() * scale.double()[:, None], want, 2.0 ** -4 + F32_WORK, 2.0 ** -10 * scale.double()[:, None] * (1 + F32_WORK))
    assert float(q.float().abs().max()) <= 448
    if rows > 1:
        assert bool((q[1:].float().abs().amax(-1) == 448).all())
    if residual:
        assert len(out) == 3
        _close(out[2], t, _half_step(dtype) + 2.0 ** -24, 2.0 ** -24)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, dim", [(1, 64), (3, 7), (700, 72), (33, 1001), (257, 2048), (1300, 1000), (65, 8192),
                                       (5, 16384), (4, 6000), (3, 5003), (1, 1)])
@pytest.mark.parametrize("residual", [False, True])
def test_gradients_against_the_formula(rows, dim, dtype, residual):
    dtype = DTYPES[dtype]
    x, r, w, dy, ds = _inputs(rows, dim, dtype, residual)
    leaves = [x.requires_grad_(), *([r.requires_grad_()] if residual else []), w.requires_grad_()]
    out = layers.rms_norm(x, w, residual=r, eps=EPS)
    outs, cots = (list(out), [dy, ds]) if residual else ([out], [dy])
    got = torch.autograd.grad(outs, leaves, cots)
    wide = [leaf.detach().double().requires_grad_() for leaf in leaves]
    t, y = _reference(wide[0], wide[1] if residual else None, wide[-1])
    want = torch.autograd.grad([y, t] if residual else [y], wide, [c.double() for c in cots])
    t, w64 = t.detach(), w.detach().double()
    rstd = 1 / torch.sqrt(t.square().mean(-1, keepdim=True) + EPS)
    n, dn = t * rstd, dy.double() * w64
    off = 4 * F32_WORK * rstd * (dn.abs() + n.abs() * (dn * n).abs().mean(-1, keepdim=True))
    for g, wt in zip(got[:-1], want[:-1]):
        assert g.dtype == dtype
        _close(g, wt, _half_step(dtype) + 2.0 ** -23, off + 2.0 ** -24)
    _close(got[-1], want[-1], 0.0, (2 * F32_WORK + rows * 2.0 ** -24) * (dy.double() * n).abs().sum(0))
    if residual:
        assert bool((got[0] == got[1]).all())


@pytest.mark.parametrize("rows, dim", [(4, 64), (3, 33)])
def test_gradients_against_differences(rows, dim):
    x, r, w, dy, ds = _inputs(rows, dim, torch.float32, True, seed=3)
    leaves = [x.requires_grad_(), r.requires_grad_(), w.requires_grad_()]
    got = torch.autograd.grad(list(layers.rms_norm(x, w, residual=r, eps=EPS)), leaves, [dy, ds])
    h = 2.0 ** -7
    for k, leaf in enumerate(leaves):
        gen = torch.Generator(device="cuda").manual_seed(k)
        d = torch.randn(leaf.shape, generator=gen, device="cuda")

        def loss(s):
            args = [v.detach() + (s * d if j == k else 0) for j, v in enumerate(leaves)]
            y, t = layers.rms_norm(args[0], args[2], residual=args[1], eps=EPS)
            return float((y.double() * dy.double()).sum() + (t.double() * ds.double()).sum())

        slope = (loss(h) - loss(-h)) / (2 * h)
        # two losses, each sum of values off by F32_WORK, over 2 h; the third derivative adds h^2 / 6 of values of order one
        # (rows of norm about 3 sqrt(dim) against steps of norm sqrt(dim): a hundredth of the slope's terms at most)
        size = float((dy.double().abs() * 4).sum() + (ds.double().abs() * 12).sum())
        assert abs(slope - float((got[k].double() * d.double()).sum())) <= size * (F32_WORK / h + h * h)


def test_only_what_is_asked_for():
    x, r, w, dy, ds = _inputs(9, 72, torch.bfloat16, True)
    y, stream = layers.rms_norm(x.requires_grad_(), w, residual=r)
    g, = torch.autograd.grad([stream], [x], [ds], retain_graph=True)  # the norm itself unused
    assert bool((g == ds).all())
    g, = torch.autograd.grad([y], [x], [dy])
    assert g.shape == x.shape
    x.requires_grad_(False)
    y, stream = layers.rms_norm(x, w.requires_grad_(), residual=r)
    g, = torch.autograd.grad([y], [w], [dy])
    assert g.shape == w.shape and not stream.requires_grad


def test_shapes_strides_and_empty():
    x, r, w, _, _ = _inputs(24, 96, torch.float16, True)
    want = layers.rms_norm(x, w, residual=r)
    got = layers.rms_norm(x.view(2, 3, 4, 96), w, residual=r.view(2, 3, 4, 96))
    for a, b in zip(got, want):
        assert a.shape == (2, 3, 4, 96) and bool((a.view(24, 96) == b).all())
    wide = torch.zeros(24, 200, dtype=torch.float16, device="cuda")
    wide[:, 3:99] = x  # rows that lie apart and start anywhere
    assert bool((layers.rms_norm(wide[:, 3:99], w) == layers.rms_norm(x, w)).all())
    odd = torch.zeros(24 * 96 + 1, dtype=torch.float16, device="cuda")[1:].view(24, 96).copy_(x)  # not on 16 bytes
    assert bool((layers.rms_norm(odd, w) == layers.rms_norm(x, w)).all())
    assert bool((layers.rms_norm(x[3], w) == layers.rms_norm(x, w)[3]).all())
    q, s = layers.rms_norm(x[3], w, out_dtype=torch.float8_e4m3fn)
    assert q.shape == (96,) and s.shape == ()
    assert layers.rms_norm(x[:0], w).shape == (0, 96)
    q, s, t = layers.rms_norm(x[:0], w, residual=r[:0], out_dtype=torch.float8_e4m3fn)
    assert q.shape == t.shape == (0, 96) and s.shape == (0,)
    e = x[:0].detach().requires_grad_()
    wg = w.detach().requires_grad_()
    ge, gw = torch.autograd.grad(layers.rms_norm(e, wg).sum(), [e, wg])
    assert ge.shape == (0, 96) and not bool(gw.any())


def test_infinities_and_nan_stay_in_their_rows():
    x, _, w, _, _ = _inputs(6, 128, torch.bfloat16, False)
    clean = layers.rms_norm(x, w)
    bad = x.clone()
    bad[1, 5], bad[3, 0], bad[4, 127] = float("nan"), float("inf"), float("-inf")
    y = layers.rms_norm(bad, w)
    assert bool((y[[0, 2, 5]] == clean[[0, 2, 5]]).all()) and bool(y[1].isnan().all())
    assert bool(y[3, 0].isnan()) and not bool(y[3, 1:].any())  # inf / inf, and all others over an infinite norm
    q, scale = layers.rms_norm(bad, w, out_dtype=torch.float8_e4m3fn)
    qc, sc = layers.rms_norm(x, w, out_dtype=torch.float8_e4m3fn)
    assert bool((q[[0, 2, 5]].float() == qc[[0, 2, 5]].float()).all()) and bool((scale[[0, 2, 5]] == sc[[0, 2, 5]]).all())
    assert bool(scale[[1, 3, 4]].isnan().all())


def test_same_bits_every_time():
    x, r, w, dy, ds = _inputs(3000, 1000, torch.bfloat16, True)
    leaves = [x.requires_grad_(), r.requires_grad_(), w.requires_grad_()]
    runs = [torch.autograd.grad(list(layers.rms_norm(x, w, residual=r)), leaves, [dy, ds]) for _ in range(3)]
    for other in runs[1:]:
        assert all(bool((a == b).all()) for a, b in zip(runs[0], other))


def test_refusals():
    x, r, w, _, _ = _inputs(4, 64, torch.bfloat16, True)
    for kw, text in ((dict(residual=r.float()), "residual"), (dict(residual=r[:2]), "residual"),
                     (dict(residual=r.cpu()), "residual"), (dict(out_dtype=torch.float16), "out_dtype")):
        with pytest.raises(ValueError, match=text):
            layers.rms_norm(x, w, **kw)
    with pytest.raises(ValueError, match="weight"):
        layers.rms_norm(x, w[:32])
    with pytest.raises(ValueError, match="weight"):
        layers.rms_norm(x, w.cpu())
    with pytest.raises(ValueError, match="dtype"):
        layers.rms_norm(x.double(), w)
    with pytest.raises(ValueError, match="16384"):
        layers.rms_norm(torch.zeros(2, 16392, device="cuda"), torch.ones(16392, device="cuda"))
    with pytest.raises(ValueError, match="no gradient"):
        layers.rms_norm(x.requires_grad_(), w, out_dtype=torch.float8_e4m3fn)
    with torch.no_grad():
        layers.rms_norm(x, w, out_dtype=torch.float8_e4m3fn)
