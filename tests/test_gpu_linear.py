"""``layers.linear`` and ``layers.gated_linear`` against their definitions in 64 bits: both kernels (few tokens, any number),
odd sizes, strides, activations, bias and residual, e4m3 operands, gradients against the formula's and against differences."""

import math

import pytest
import torch

from jax_linear_attention_b200 import layers

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
TINY = 2.0 ** -24  # float16 below its normal numbers


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _act64(name, z):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "sigmoid":
        return torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _inputs(rows, depth, out, dtype, *, bias=False, residual=False, gated=False, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = {"x": _randn(gen, rows, depth).to(dtype), "w": (_randn(gen, out, depth) / math.sqrt(depth)).to(dtype)}
    if gated:
        t["up"] = (_randn(gen, out, depth) / math.sqrt(depth)).to(dtype)
    t["b"] = 0.5 * _randn(gen, out) if bias else None
    t["r"] = _randn(gen, rows, out).to(dtype) if residual else None
    t["dy"] = _randn(gen, rows, out).to(dtype)
    return t


def _close(got, want, bound):
    err = (got.double() - want).abs() - bound
    assert bool((err <= 0).all()), float(err.max())


def _sum_bound(a, b, depth):
    """What float32 sums of `depth` products may be off by, each addition rounding (or cutting off) to 2^-23 of the terms'
    sum so far at most: a @ b of absolute values."""
    return depth * 2.0 ** -23 * (a.abs() @ b.abs())


# An activation in float32: its exponential and reciprocal are off by 2^-21 relative, so is its value, of at most |z| + 1.
ACT = 2.0 ** -20
SLOPE = 1.2  # the largest |act'|


def _check_linear(t, act, y, dtype):
    x, w = t["x"].double(), t["w"].double()
    z = x @ w.t() + (0 if t["b"] is None else t["b"].double())
    want = _act64(act, z) + (0 if t["r"] is None else t["r"].double())
    off = SLOPE * (_sum_bound(x, w.t(), x.shape[1]) + 2.0 ** -23 * z.abs()) + ACT * (1 + z.abs())
    _close(y, want, (off + _half_step(dtype) * want.abs()) * (1 + 2.0 ** -7) + TINY)


SIZES = [(1, 64, 64), (1, 8, 8), (3, 72, 136), (16, 2048, 256), (17, 200, 1000), (33, 512, 72), (100, 328, 264), (128, 4096, 128),
         (130, 64, 640), (256, 136, 384), (257, 8, 200), (300, 200, 264), (700, 520, 1000), (1003, 2048, 512), (2049, 72, 8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, depth, out", SIZES)
def test_linear_forward(rows, depth, out, dtype):
    dtype = DTYPES[dtype]
    t = _inputs(rows, depth, out, dtype)
    y = layers.linear(t["x"], t["w"])
    assert y.dtype == dtype and y.shape == (rows, out)
    _check_linear(t, None, y, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", [None, "silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("bias, residual", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("rows, depth, out", [(5, 136, 200), (90, 256, 104), (600, 136, 328)])
def test_linear_epilogue(rows, depth, out, act, bias, residual, dtype):
    dtype = DTYPES[dtype]
    t = _inputs(rows, depth, out, dtype, bias=bias, residual=residual, seed=1)
    _check_linear(t, act, layers.linear(t["x"], t["w"], t["b"], activation=act, residual=t["r"]), dtype)


def _check_linear_gradients(rows, depth, out, dtype, act, bias, residual, seed=2):
    t = _inputs(rows, depth, out, dtype, bias=bias, residual=residual, seed=seed)
    names = [n for n in ("x", "w", "b", "r") if t[n] is not None]
    leaves = [t[n].requires_grad_() for n in names]
    y = layers.linear(t["x"], t["w"], t["b"], activation=act, residual=t["r"])
    got = dict(zip(names, torch.autograd.grad(y, leaves, t["dy"])))
    wide = {n: t[n].detach().double().requires_grad_() for n in names}
    x, w = wide["x"], wide["w"]
    z = x @ w.t() + (wide["b"] if bias else 0)
    ref = _act64(act, z) + (wide["r"] if residual else 0)
    want = dict(zip(names, torch.autograd.grad(ref, [wide[n] for n in names], t["dy"].double(), retain_graph=True)))
    dz, = torch.autograd.grad(ref, [z], t["dy"].double())
    x, w, z = x.detach(), w.detach(), z.detach()
    # dz: z is off by its sum's error (|act''| <= 1.2), the slope by ACT; its rounding where there is an activation
    dy = t["dy"].double().abs()
    dz_off = 0 * dz
    if act:
        dz_off = dy * (1.2 * (_sum_bound(x, w.t(), depth) + 2.0 ** -23 * z.abs()) + ACT * (1 + z.abs()))
    dz_off16 = dz_off + ((_half_step(dtype) * (dz.abs() + dz_off) + TINY) if act else 0)
    step = _half_step(dtype)
    for name, off in (("x", dz_off16 @ w.abs() + _sum_bound(dz, w, out)), ("w", dz_off16.t() @ x.abs() + _sum_bound(dz.t(), x, rows))):
        assert got[name].dtype == dtype and got[name].shape == t[name].shape
        _close(got[name], want[name], (off + step * want[name].abs()) * (1 + 2.0 ** -7) + TINY)
    if bias:
        assert got["b"].dtype == torch.float32
        _close(got["b"], want["b"], dz_off.sum(0) + rows * 2.0 ** -23 * dz.abs().sum(0))
    if residual:
        assert bool((got["r"] == t["dy"]).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, depth, out", [(1, 64, 72), (1, 8, 8), (17, 200, 136), (100, 128, 520), (256, 72, 64),
                                              (300, 264, 200), (1003, 512, 328), (2500, 8, 16)])
@pytest.mark.parametrize("act, bias, residual", [(None, False, False), (None, True, True), ("silu", False, True),
                                                 ("sigmoid", True, False), ("gelu", True, True)])
def test_linear_gradients(rows, depth, out, dtype, act, bias, residual):
    _check_linear_gradients(rows, depth, out, DTYPES[dtype], act, bias, residual)


@pytest.mark.parametrize("rows, depth, out", [(1, 1, 1), (5, 7, 3), (30, 64, 6), (300, 100, 12), (130, 33, 257), (9000, 70, 50)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_any_width(rows, depth, out, dtype):
    dtype = DTYPES[dtype]
    t = _inputs(rows, depth, out, dtype, bias=True, residual=True, seed=9)
    y = layers.linear(t["x"], t["w"], t["b"], activation="silu", residual=t["r"])
    assert y.shape == (rows, out) and y.is_contiguous()
    _check_linear(t, "silu", y, dtype)
    _check_linear_gradients(rows, depth, out, dtype, "gelu", True, True)
    _check_gated(rows, depth, out, dtype, "silu", True)


# Every kernel and tile width: few tokens (16, 32, 64 or 128 of them a block), pairs of CTAs (128 or 256 columns a tile, one
# tile a pair and several).
KERNELS = [(5, 2048, 136), (20, 520, 200), (50, 1000, 72), (100, 2048, 264), (100, 72, 2000), (1500, 4096, 24), (2100, 72, 56),
           (8300, 72, 56), (8300, 264, 72), (8300, 136, 136), (5000, 72, 1000), (2100, 520, 1000), (8300, 72, 2600), (9400, 136, 264),
           (18900, 72, 256)]


@pytest.mark.parametrize("rows, depth, out", KERNELS)
def test_every_kernel(rows, depth, out):
    t = _inputs(rows, depth, out, torch.bfloat16, bias=True, residual=True)
    _check_linear(t, "silu", layers.linear(t["x"], t["w"], t["b"], activation="silu", residual=t["r"]), torch.bfloat16)
    _check_linear_gradients(rows, depth, out, torch.bfloat16, "silu", True, True)
    _check_linear_gradients(rows, depth, out, torch.float16, None, False, False)


def test_weight_gradients_of_many_tiles():
    _check_linear_gradients(100, 1792, 2560, torch.float16, None, False, False)  # 70 tiles
    _check_linear_gradients(100, 2048, 4096, torch.bfloat16, None, False, False)  # 128


def _gated64(x, w, up, act):
    return _act64(act, x @ w.t()) * (x @ up.t())


def _check_gated(rows, depth, out, dtype, act, grads, seed=3):
    t = _inputs(rows, depth, out, dtype, gated=True, seed=seed)
    names = ["x", "w", "up"]
    leaves = [t[n].requires_grad_(grads) for n in names]
    y = layers.gated_linear(*leaves, activation=act)
    x, w, up = (v.detach().double().requires_grad_(grads) for v in leaves)
    g, u = x @ w.t(), x @ up.t()
    ref = _act64(act, g) * u
    xd, wd, ud, gd, vd = (v.detach() for v in (x, w, up, g, u))
    g_off, u_off = (_sum_bound(xd, m.t(), depth) + 2.0 ** -23 * v.abs() for m, v in ((wd, gd), (ud, vd)))
    a, step = _act64(act, gd).abs(), _half_step(dtype)
    a_off = SLOPE * g_off + ACT * (1 + gd.abs())
    h_off = a_off * (vd.abs() + u_off) + a * u_off
    want = ref.detach()
    _close(y, want, (h_off + step * want.abs()) * (1 + 2.0 ** -7) + TINY)
    if not grads:
        return
    dy = t["dy"].double()
    got = torch.autograd.grad(y, leaves, t["dy"])
    wanted = torch.autograd.grad(ref, [x, w, up], dy, retain_graph=True)
    dg, du = torch.autograd.grad(ref, [g, u], dy)
    slope_off = 1.2 * g_off + ACT * (1 + gd.abs())
    dg_off = dy.abs() * (slope_off * (vd.abs() + u_off) + SLOPE * u_off)
    du_off = dy.abs() * a_off
    dg_off, du_off = (o + step * (d.abs() + o) + TINY for o, d in ((dg_off, dg), (du_off, du)))
    offs = (dg_off @ wd.abs() + du_off @ ud.abs() + _sum_bound(torch.cat([dg, du], 1), torch.cat([wd, ud], 0), 2 * out),
            dg_off.t() @ xd.abs() + _sum_bound(dg.t(), xd, rows), du_off.t() @ xd.abs() + _sum_bound(du.t(), xd, rows))
    for g_, w_, o in zip(got, wanted, offs):
        assert g_.dtype == dtype
        _close(g_, w_, (o + step * w_.abs()) * (1 + 2.0 ** -7) + TINY)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, depth, out", SIZES)
def test_gated_forward(rows, depth, out, dtype):
    _check_gated(rows, depth, out, DTYPES[dtype], "silu", False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("rows, depth, out", [(1, 64, 72), (17, 200, 136), (100, 128, 264), (300, 264, 200), (1003, 512, 328)])
def test_gated_gradients(rows, depth, out, act, dtype):
    _check_gated(rows, depth, out, DTYPES[dtype], act, True)


@pytest.mark.parametrize("rows, depth, out", KERNELS)
def test_gated_every_kernel(rows, depth, out):
    _check_gated(rows, depth, out, torch.bfloat16, "silu", True)


def test_gated_weight_gradients_of_many_tiles():
    _check_gated(70, 1792, 1280, torch.float16, "silu", True)  # dWg and dWu: 2 x 5 x 7 tiles


def _e4m3(x):
    scale = x.abs().amax(-1).clamp_min(1e-12) / 448
    return (x / scale[:, None]).to(torch.float8_e4m3fn), scale


@pytest.mark.parametrize("rows, depth, out", [(1, 64, 64), (1, 16, 8), (5, 2048, 136), (33, 208, 1000), (100, 4096, 72),
                                              (200, 144, 264), (300, 16, 200), (1003, 1024, 520), (18900, 80, 256),
                                              (20, 4096, 136), (60, 4096, 136), (3, 7, 5), (300, 100, 12), (8300, 80, 56), (8300, 80, 200), (5000, 144, 1000), (9400, 80, 264)])
@pytest.mark.parametrize("out_dtype", DTYPES)
def test_e4m3(rows, depth, out, out_dtype):
    dtype = DTYPES[out_dtype]
    gen = torch.Generator(device="cuda").manual_seed(4)
    x, xs = _e4m3(_randn(gen, rows, depth))
    (w, ws), (up, us) = (_e4m3(_randn(gen, out, depth) / math.sqrt(depth)) for _ in range(2))
    b, r = 0.5 * _randn(gen, out), _randn(gen, rows, out).to(dtype)
    xd, wd, ud = (q.double() * s.double()[:, None] for q, s in ((x, xs), (w, ws), (up, us)))
    g, u = xd @ wd.t(), xd @ ud.t()
    # e4m3 products are exact in float32; their sums are taken to at least 2^-13 of the largest term in each of the
    # depth / 32 instructions' additions (the 8-bit kind need not keep all of float32's bits), then the scales round
    g_off, u_off = ((2.0 ** -13 + depth * 2.0 ** -23) * (xd.abs() @ m.abs().t()) for m in (wd, ud))
    y = layers.linear(x, w, b, activation="silu", residual=r, x_scale=xs, weight_scale=ws, out_dtype=dtype)
    assert y.dtype == dtype
    z = g + b.double()
    want = _act64("silu", z) + r.double()
    _close(y, want, (SLOPE * g_off + ACT * (1 + z.abs()) + _half_step(dtype) * want.abs()) * (1 + 2.0 ** -7) + TINY)
    h = layers.gated_linear(x, w, up, x_scale=xs, gate_scale=ws, up_scale=us, out_dtype=dtype)
    a = _act64("silu", g)
    want = a * u
    off = (SLOPE * g_off + ACT * (1 + g.abs())) * (u.abs() + u_off) + a.abs() * u_off
    _close(h, want, (off + _half_step(dtype) * want.abs()) * (1 + 2.0 ** -7) + TINY)


@pytest.mark.parametrize("rows", [12, 400, 8300])
def test_gradients_against_differences(rows):
    t = _inputs(rows, 64, 72, torch.float16, gated=True, seed=6)
    leaves = [t[n].requires_grad_() for n in ("x", "w", "up")]
    got = torch.autograd.grad(layers.gated_linear(*leaves), leaves, t["dy"])
    wide = [v.detach().double() for v in leaves]
    for k in range(3):
        d = torch.randn(wide[k].shape, generator=torch.Generator(device="cuda").manual_seed(k), device="cuda").double()

        def loss(s):
            return float((_gated64(*(v + (s * d if j == k else 0) for j, v in enumerate(wide)), "silu") * t["dy"].double()).sum())

        h = 2.0 ** -14  # truncation h^2, rounding 2^-53 / h: both far below what follows
        slope = (loss(h) - loss(-h)) / (2 * h)
        # every element of a gradient is off by half a step of itself and of the dg and du it sums (at most all of one sign)
        size = float((got[k].double().abs() * d.abs()).sum())
        assert abs(slope - float((got[k].double() * d).sum())) <= 4 * 2.0 ** -11 * size


def test_shapes_strides_and_slices():
    t = _inputs(24, 64, 72, torch.bfloat16, bias=True, residual=True)
    want = layers.linear(t["x"], t["w"], t["b"], residual=t["r"])
    got = layers.linear(t["x"].view(2, 3, 4, 64), t["w"], t["b"], residual=t["r"].view(2, 3, 4, 72))
    assert got.shape == (2, 3, 4, 72) and bool((got.view(24, 72) == want).all())
    assert bool((layers.linear(t["x"][5], t["w"], t["b"], residual=t["r"][5]) == want[5]).all())
    wide = torch.full((24, 160), 7.0, dtype=torch.bfloat16, device="cuda")
    for start in (0, 16, 3):  # rows that lie apart: read in place, in place, copied (not on 16 bytes)
        wide[:, start:start + 64] = t["x"]
        assert bool((layers.linear(wide[:, start:start + 64], t["w"], t["b"], residual=t["r"]) == want).all())
    assert bool((layers.linear(t["x"], t["w"].t().contiguous().t(), t["b"], residual=t["r"]) == want).all())
    same = t["x"][:1].expand(24, 64)
    assert bool((layers.linear(same, t["w"]) == layers.linear(same.contiguous(), t["w"])).all())
    b = torch.cat([t["b"][:1], t["b"]])[1:]  # not on 16 bytes
    assert bool((layers.linear(t["x"], t["w"], b, residual=t["r"]) == want).all())


@pytest.mark.parametrize("rows", [20, 400, 8300])
def test_gradients_of_slices_and_broadcasts(rows):
    t = _inputs(rows, 64, 72, torch.float16, gated=True)
    wide = torch.randn(rows, 200, device="cuda").half()
    wide[:, 8:72] = t["x"]
    wide.requires_grad_()
    x = t["x"].clone().requires_grad_()
    for fn, w in ((lambda v, *m: layers.linear(v, m[0], activation="silu"), (t["w"],)),
                  (lambda v, *m: layers.gated_linear(v, *m), (t["w"], t["up"]))):
        w = [m.clone().requires_grad_() for m in w]
        a = torch.autograd.grad(fn(wide[:, 8:72], *w), [wide, *w], t["dy"])
        b = torch.autograd.grad(fn(x, *w), [x, *w], t["dy"])
        assert bool((a[0][:, 8:72] == b[0]).all()) and not bool(a[0][:, 72:].any())
        assert all(bool((p == q).all()) for p, q in zip(a[1:], b[1:]))
        # a gradient that is one number for all outputs comes as an expanded tensor
        one = torch.autograd.grad(fn(x, *w).sum(), [x, *w])
        ones = torch.autograd.grad(fn(x, *w), [x, *w], torch.ones_like(t["dy"]))
        assert all(bool((p == q).all()) for p, q in zip(one, ones))


def test_no_rows():
    t = _inputs(4, 64, 72, torch.bfloat16, bias=True, gated=True)
    x = t["x"][:0].requires_grad_()
    w, up, b = (t[n].requires_grad_() for n in ("w", "up", "b"))
    y = layers.linear(x, w, b, activation="silu")
    assert y.shape == (0, 72)
    for g in torch.autograd.grad(y.sum(), [x, w, b]):
        assert not bool(g.any())
    h = layers.gated_linear(x, w, up)
    for g in torch.autograd.grad(h.sum(), [x, w, up]):
        assert not bool(g.any())
    q, s = torch.zeros(0, 64, device="cuda").to(torch.float8_e4m3fn), torch.zeros(0, device="cuda")
    qw, sw = _e4m3(t["w"].detach().float())
    assert layers.linear(q, qw, x_scale=s, weight_scale=sw).shape == (0, 72)
    assert layers.gated_linear(q, qw, qw, x_scale=s, gate_scale=sw, up_scale=sw).shape == (0, 72)


def test_what_lies_behind_the_rows_is_left_alone():
    for rows, depth, out in ((5, 64, 72), (130, 64, 72), (300, 64, 72), (8300, 64, 72), (8300, 64, 200)):
        t = _inputs(rows, depth, out, torch.bfloat16)
        y = layers.linear(t["x"], t["w"])
        space = torch.full((rows + 300, out), 9.0, dtype=torch.bfloat16, device="cuda")
        from jax_linear_attention_b200 import _lib
        _lib.launch("jla_linear_fwd", space.device, 0, 0, rows, depth, out, t["x"].data_ptr(), depth, t["w"].data_ptr(), None,
                    None, None, 0, None, space.data_ptr(), None)
        assert bool((space[:rows] == y).all()) and bool((space[rows:] == 9).all())


@pytest.mark.parametrize("rows", [7, 200, 600, 8300])
def test_infinities_and_nan_stay_in_their_rows(rows):
    t = _inputs(rows, 72, 72, torch.bfloat16)
    want = layers.linear(t["x"], t["w"])
    bad = t["x"].clone()
    bad[rows - 2, 71], bad[2, 0] = float("nan"), float("inf")
    got = layers.linear(bad, t["w"])
    keep = [i for i in range(rows) if i not in (2, rows - 2)]
    assert bool((got[keep] == want[keep]).all()) and bool(got[rows - 2].isnan().all()) and not bool(got[2].isfinite().any())


@pytest.mark.parametrize("rows", [20, 8300])
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_activations_far_out(rows, act):
    """Products up to 1e20, where exponentials and powers overflow: the activation is the identity or zero (or one), its slope
    one or zero."""
    x = torch.zeros(rows, 64, device="cuda", dtype=torch.bfloat16)
    size = torch.logspace(2, 20, rows, device="cuda") * (1 - 2 * (torch.arange(rows, device="cuda") % 2))
    x[:, 0] = size.bfloat16()
    w = torch.zeros(72, 64, device="cuda", dtype=torch.bfloat16)
    w[:, 0] = 1
    x.requires_grad_(), w.requires_grad_()
    z = x.detach().float()[:, :1].expand(rows, 72)
    up = (z > 0).float()
    y = layers.linear(x, w, activation=act)
    assert bool((y.float() == (up if act == "sigmoid" else z * up)).all())
    dx, = torch.autograd.grad(y, [x], torch.ones_like(y))
    assert bool((dx[:, 0].float() == (0 * up[:, 0] if act == "sigmoid" else 72 * up[:, 0])).all()) and not bool(dx[:, 1:].any())
    h = layers.gated_linear(x, w, 2.0 ** -10 * w.detach(), activation=act)
    assert bool(h.isfinite().all() if act == "sigmoid" else (h.float()[z < 0] == 0).all())


def test_only_what_is_asked_for():
    t = _inputs(40, 64, 72, torch.bfloat16, bias=True, gated=True)
    for name in ("x", "w", "b"):
        leaf = t[name].detach().clone().requires_grad_()
        args = [leaf if n == name else t[n].detach() for n in ("x", "w", "b")]
        full = [t[n].detach().clone().requires_grad_() for n in ("x", "w", "b")]
        want = torch.autograd.grad(layers.linear(*full, activation="gelu"), full, t["dy"])[("x", "w", "b").index(name)]
        got, = torch.autograd.grad(layers.linear(*args, activation="gelu"), [leaf], t["dy"])
        assert bool((got == want).all())
    for name in ("x", "w", "up"):
        leaf = t[name].detach().clone().requires_grad_()
        args = [leaf if n == name else t[n].detach() for n in ("x", "w", "up")]
        full = [t[n].detach().clone().requires_grad_() for n in ("x", "w", "up")]
        want = torch.autograd.grad(layers.gated_linear(*full), full, t["dy"])[("x", "w", "up").index(name)]
        got, = torch.autograd.grad(layers.gated_linear(*args), [leaf], t["dy"])
        assert bool((got == want).all())


def test_one_dimension_and_other_biases():
    t = _inputs(3, 64, 72, torch.bfloat16, bias=True, residual=True)
    q, s = _e4m3(t["x"].float())
    qw, sw = _e4m3(t["w"].float())
    want = layers.linear(q, qw, x_scale=s, weight_scale=sw)
    assert bool((layers.linear(q[1], qw, x_scale=s[1], weight_scale=sw) == want[1]).all())
    b16 = t["b"].bfloat16().requires_grad_()  # a bias in 16 bits is used as it is, and so is its gradient's type
    y = layers.linear(t["x"], t["w"], b16)
    assert bool((y == layers.linear(t["x"], t["w"], b16.detach().float())).all())
    g, = torch.autograd.grad(y, [b16], t["dy"])
    assert g.dtype == torch.bfloat16
    _close(g, t["dy"].double().sum(0), 2.0 ** -8 * t["dy"].double().sum(0).abs() + 1e-5)
    r = t["r"].clone().requires_grad_()  # the residual alone
    g, = torch.autograd.grad(layers.linear(t["x"], t["w"], t["b"], residual=r, activation="silu"), [r], t["dy"])
    assert bool((g == t["dy"]).all())
    g, = torch.autograd.grad(layers.linear(t["x"], t["w"], residual=r), [r], t["dy"])
    assert bool((g == t["dy"]).all())


def test_refusals():
    t = _inputs(4, 64, 72, torch.bfloat16, bias=True, residual=True, gated=True)
    x, w, up, b, r = (t[n] for n in ("x", "w", "up", "b", "r"))
    q, s = _e4m3(x.float())
    qw, sw = _e4m3(w.float())
    for call, text in (
            (lambda: layers.linear(x, w.half()), "share one of"), (lambda: layers.linear(x.float(), w.float()), "share one of"),
            (lambda: layers.linear(x[:, :56], w), "expected x"), (lambda: layers.linear(x[:, :0], w[:, :0]), "features"),
            (lambda: layers.linear(x, w[:0]), "features"), (lambda: layers.linear(x, w, b[:64]), "bias"),
            (lambda: layers.linear(x, w, b.cpu()), "bias"), (lambda: layers.linear(x, w, residual=r.float()), "residual"),
            (lambda: layers.linear(x, w, residual=r[:1]), "residual"), (lambda: layers.linear(x, w, x_scale=s), "scales"),
            (lambda: layers.linear(x, w, out_dtype=torch.float16), "out_dtype"), (lambda: layers.linear(q, qw), "x_scale"),
            (lambda: layers.linear(q, qw, x_scale=s, weight_scale=sw[:5]), "weight scale"),
            (lambda: layers.linear(q, qw, x_scale=s.double(), weight_scale=sw), "x_scale"),
            (lambda: layers.linear(q, qw, x_scale=s, weight_scale=sw, out_dtype=torch.float32), "out_dtype"),
            (lambda: layers.linear(q, qw, x_scale=s, weight_scale=sw, bias=b.clone().requires_grad_()), "no gradient"),
            (lambda: layers.gated_linear(x, w, up[:64]), "expected x"), (lambda: layers.gated_linear(x, w, up.half()), "share one of"),
            (lambda: layers.gated_linear(q, qw, qw, x_scale=s, gate_scale=sw), "weight scale"),
            (lambda: layers.gated_linear(x, w, up.cpu()), "CUDA tensor")):
        with pytest.raises(ValueError, match=text):
            call()
