"""Cases of the operators around a mixer: the residual stream's RMS norm, the projections, the gated feed-forward block.

* ``norm``: ``layers.rms_norm`` with the residual's addition, its gradient, its output in e4m3 with one scale a row;
* ``linear``: ``layers.linear``, a product with bias, activation and residual, its gradients, its form for e4m3 operands;
* ``gated``: ``layers.gated_linear``, both projections of a gated feed-forward block, its gradients, its form for e4m3.

The model width is 2048 (16 heads of 128, the widths of the framework's own workloads), the inner width of a Mamba-2 layer
4096 (64 heads of 64), its input projection 2 * 4096 + 2 * 128 + 64 = 8512 wide; 16384 tokens are a batch of 8 x 2048.

``own`` false: the plain forms, in 32 bits and rounded once. ``own`` true: the calls that a user makes.
"""

import math

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # one decoding step of one sequence: the norm in front of a mixer
        dict(name="norm 1 x 2048", op="norm", rows=1, dim=2048, dtype="bf16", out="same", residual=True, train=False),
        # a prompt's tokens on their way into 8-bit projections of an inner width of 4096
        dict(name="norm 5003 x 4096 to e4m3", op="norm", rows=5003, dim=4096, dtype="f16", out="e4m3", residual=True,
             train=False),
        # the pre-norm of a training step, 8 x 2048 tokens
        dict(name="norm 16384 x 2048 training", op="norm", rows=16384, dim=2048, dtype="bf16", out="same", residual=True,
             train=True),
        # a small float32 model of an odd width
        dict(name="norm 1111 x 1001 f32 training", op="norm", rows=1111, dim=1001, dtype="f32", out="same", residual=False,
             train=True),
        # one decoding step: the input projection of a Mamba-2 layer
        dict(name="linear 1 x 2048 x 8512", op="linear", rows=1, inner=2048, outer=8512, dtype="bf16", bias=True, act="none",
             residual=False, train=False),
        # a decoding step of 33 sequences in 8 bits: the output projection into the residual stream
        dict(name="linear 33 x 4096 x 2048 e4m3", op="linear", rows=33, inner=4096, outer=2048, dtype="e4m3", bias=False,
             act="none", residual=True, train=False),
        # a prompt of 1003 tokens: q, k and v of 2048 channels each
        dict(name="linear 1003 x 2048 x 6144", op="linear", rows=1003, inner=2048, outer=6144, dtype="f16", bias=True,
             act="silu", residual=False, train=False),
        # training: the erase or write gates of a mixer with gates per channel
        dict(name="linear 4096 x 2048 x 2048 training", op="linear", rows=4096, inner=2048, outer=2048, dtype="f16",
             bias=True, act="sigmoid", residual=False, train=True),
        # training: the output projection of a Mamba-2 layer, 8 x 2048 tokens
        dict(name="linear 16384 x 4096 x 2048 training", op="linear", rows=16384, inner=4096, outer=2048, dtype="bf16",
             bias=False, act="none", residual=True, train=True),
        # a decoding step of four sequences
        dict(name="gated 4 x 2048 x 5632", op="gated", rows=4, inner=2048, outer=5632, dtype="bf16", act="silu",
             train=False),
        # a ragged prefill in 8 bits
        dict(name="gated 5003 x 2048 x 5632 e4m3", op="gated", rows=5003, inner=2048, outer=5632, dtype="e4m3", act="silu",
             train=False),
        # the largest: a training step's feed-forward block, 8 x 2048 tokens
        dict(name="gated 16384 x 2048 x 5632 training", op="gated", rows=16384, inner=2048, outer=5632, dtype="bf16",
             act="silu", train=True),
    ]


LARGEST = 3 * 4 * 16384 * 2048 * 5632  # flops of the largest listed case


def _log(rng, low, high, step=1):
    """A multiple of ``step`` between ``low`` and ``high``, evenly spread over the logarithm."""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + step))) // step * step)))


def draw(rng):
    op = rng.choice(["norm", "linear", "gated"])
    if op == "norm":
        dtype = rng.choice(["bf16", "f16", "f32"])
        train = rng.random() < 0.4
        out = "e4m3" if not train and rng.random() < 0.5 else "same"
        dim = _log(rng, 64, 8192, rng.choice([1, 8, 64]))
        return dict(op=op, rows=min(_log(rng, 1, 16384), 16384 * 2048 // dim), dim=dim, dtype=dtype, out=out,
                    residual=rng.random() < 0.7, train=train)
    dtype = rng.choice(["bf16", "f16", "e4m3"])
    train = dtype != "e4m3" and rng.random() < 0.5
    inner, outer = _log(rng, 64, 8192, 16), _log(rng, 64, 8512, rng.choice([8, 64]))
    flops = 2 * inner * outer * (3 if train else 1) * (2 if op == "gated" else 1)
    rows = min(_log(rng, 1, 16384), LARGEST // flops)
    if op == "gated":
        return dict(op=op, rows=rows, inner=inner, outer=outer, dtype=dtype, act=rng.choice(["silu", "gelu", "sigmoid"]),
                    train=train)
    return dict(op=op, rows=rows, inner=inner, outer=outer, dtype=dtype, bias=rng.random() < 0.5,
                act=rng.choice(["none", "none", "silu", "gelu", "sigmoid"]), residual=rng.random() < 0.5, train=train)


def _to_e4m3(x):
    """``(codes, scale)`` of the rows of ``x``, as a program lays out 8-bit weights once."""
    scale = x.abs().amax(-1).clamp_min(1e-12) / E4M3_MAX
    return (x / scale[:, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s, train = dict(case), case["train"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        wide = 1 + 7 * (torch.rand(dim, generator=gen, device="cuda") < 0.02)  # a stream has a few loud channels
        s["x"] = normal(rows, dim).to(dtype).requires_grad_(train)
        s["residual"] = (2 * normal(rows, dim) * wide).to(dtype).requires_grad_(train) if case["residual"] else None
        s["weight"] = (1 + 0.2 * normal(dim)).requires_grad_(train)
        if train:
            s["dy"] = normal(rows, dim).to(dtype)
            s["dstream"] = normal(rows, dim).to(dtype) if case["residual"] else None
        return s
    rows, inner, outer = case["rows"], case["inner"], case["outer"]
    out = torch.bfloat16 if case["dtype"] == "e4m3" else dtype

    def operand(x):
        return _to_e4m3(x) if case["dtype"] == "e4m3" else (x.to(dtype).requires_grad_(train), None)

    s["x"], s["x_scale"] = operand(normal(rows, inner))
    s["w"], s["w_scale"] = operand(normal(outer, inner) / math.sqrt(inner))
    if case["op"] == "gated":
        s["up"], s["up_scale"] = operand(normal(outer, inner) / math.sqrt(inner))
    else:
        s["b"] = (0.2 * normal(outer)).requires_grad_(train) if case["bias"] else None
        s["residual"] = normal(rows, outer).to(out).requires_grad_(train) if case["residual"] else None
    if train:
        s["dy"] = normal(rows, outer).to(out)
    return s


def run(state):
    s = state
    if own:
        return _own_run(s)
    return {"norm": _plain_norm, "linear": _plain_linear, "gated": _plain_gated}[s["op"]](s)


# ---- the framework's calls ----------------------------------------------------------------------------------------------


def _own_run(s):
    from jax_linear_attention_b200 import layers

    act = None if s.get("act") == "none" else s.get("act")
    if s["op"] == "norm":
        out = layers.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS,
                              out_dtype=torch.float8_e4m3fn if s["out"] == "e4m3" else None)
        out = list(out) if isinstance(out, tuple) else [out]
        if s["train"]:
            leaves = [x for x in (s["x"], s["residual"], s["weight"]) if x is not None]
            return out + list(torch.autograd.grad(out, leaves, [x for x in (s["dy"], s["dstream"]) if x is not None]))
        return out
    if s["op"] == "linear":
        y = layers.linear(s["x"], s["w"], s["b"], activation=act, residual=s["residual"], x_scale=s["x_scale"],
                          weight_scale=s["w_scale"])
        leaves = [x for x in (s["x"], s["w"], s["b"], s["residual"]) if x is not None]
    else:
        y = layers.gated_linear(s["x"], s["w"], s["up"], activation=act, x_scale=s["x_scale"], gate_scale=s["w_scale"],
                                up_scale=s["up_scale"])
        leaves = [s["x"], s["w"], s["up"]]
    if s["train"]:
        return [y, *torch.autograd.grad(y, leaves, s["dy"])]
    return [y]


# ---- plain forms: 32 bits, rounded once ---------------------------------------------------------------------------------


def _plain_norm(s):
    x, r, w = s["x"].detach(), s["residual"], s["weight"].detach()
    t = x.float() if r is None else x.float() + r.detach().float()
    rstd = (t.square().mean(-1, keepdim=True) + EPS).rsqrt()
    n = t * rstd
    y = n * w
    stream = [] if r is None else [t.to(x.dtype)]
    if s["out"] == "e4m3":
        top = y.abs().amax(-1)
        scale = torch.where(top == 0, torch.ones_like(top), top / E4M3_MAX)
        return [(y / scale[:, None]).to(torch.float8_e4m3fn), scale, *stream]
    out = [y.to(x.dtype), *stream]
    if not s["train"]:
        return out
    dy = s["dy"].float()
    dn = dy * w
    dt = rstd * (dn - n * (dn * n).mean(-1, keepdim=True))
    if r is not None:
        dt = dt + s["dstream"].float()
    dx = dt.to(x.dtype)
    return out + [dx] + ([] if r is None else [dx]) + [(dy * n).sum(0)]


def _act(name, z):
    """``(act(z), act'(z))``"""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "gelu":  # the tanh form
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    g = 1 / (1 + torch.exp(-z))
    return (g, g * (1 - g)) if name == "sigmoid" else (z * g, g * (1 + z * (1 - g)))


def _float(x, scale):
    x = x.detach().float()
    return x if scale is None else x * scale[:, None]


def _plain_linear(s):
    x, w = _float(s["x"], s["x_scale"]), _float(s["w"], s["w_scale"])
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].detach()
    y, slope = _act(s["act"], z)
    if s["residual"] is not None:
        y = y + s["residual"].detach().float()
    y = y.to(torch.bfloat16 if s["dtype"] == "e4m3" else DTYPES[s["dtype"]])
    if not s["train"]:
        return [y]
    dz = s["dy"].float() * slope
    out = [y, (dz @ w).to(y.dtype), (dz.t() @ x).to(y.dtype)]
    if s["b"] is not None:
        out.append(dz.sum(0))
    if s["residual"] is not None:
        out.append(s["dy"])
    return out


def _plain_gated(s):
    x, w, up = _float(s["x"], s["x_scale"]), _float(s["w"], s["w_scale"]), _float(s["up"], s["up_scale"])
    a, slope = _act(s["act"], x @ w.t())
    u = x @ up.t()
    y = (a * u).to(torch.bfloat16 if s["dtype"] == "e4m3" else DTYPES[s["dtype"]])
    if not s["train"]:
        return [y]
    dy = s["dy"].float()
    dg, du = dy * u * slope, dy * a
    return [y, (dg @ w + du @ up).to(y.dtype), (dg.t() @ x).to(y.dtype), (du.t() @ x).to(y.dtype)]


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

SIZE = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "norm":
        n, streams = case["rows"] * case["dim"], 2 if case["residual"] else 0  # the residual in, the new one out
        nbytes = n * size * (1 + streams) + n * (1 if case["out"] == "e4m3" else size) + 4 * case["dim"]
        if case["out"] == "e4m3":
            nbytes += 4 * case["rows"]
        if case["train"]:  # the gradients of both outputs in, one gradient (x's is the residual's) and the weight's out
            nbytes += n * size * (3 if case["residual"] else 2) + 4 * case["dim"]
        return {"bytes": nbytes, "flops": n * (16 if case["train"] else 6)}
    rows, inner, outer = case["rows"], case["inner"], case["outer"]
    out, weights = (2 if case["dtype"] == "e4m3" else size), inner * outer * (2 if case["op"] == "gated" else 1)
    nbytes = rows * inner * size + weights * size + rows * outer * out
    if case["dtype"] == "e4m3":
        nbytes += 4 * (rows + weights // inner)
    if case.get("bias"):
        nbytes += 4 * outer
    if case.get("residual"):
        nbytes += rows * outer * out
    if case["train"]:  # dy in; the gradients of x, the weights and the bias out (the residual's is dy)
        nbytes += rows * outer * out + rows * inner * size + weights * size + (4 * outer if case.get("bias") else 0)
    return {"bytes": nbytes, "flops": 2 * rows * weights * (3 if case["train"] else 1)}


# ---- 64 bits: the definitions, differentiated by torch ------------------------------------------------------------------


def _activation64(name, z):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "sigmoid":
        return torch.sigmoid(z)
    if name == "gelu":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))  # (1 + tanh t) / 2 = sigmoid(2 t)
    return z


def exact(case, seed):
    s = prepare(case, seed)

    def wide(name, scale=None):
        if s.get(name) is None:
            return None
        x = s[name].detach().double()
        return (x if s.get(scale) is None else x * s[scale].double()[:, None]).requires_grad_(case["train"])

    if case["op"] == "norm":
        x, r, w = wide("x"), wide("residual"), wide("weight")
        t = x if r is None else x + r
        y = t / torch.sqrt((t ** 2).sum(-1, keepdim=True) / case["dim"] + EPS) * w
        stream = [] if r is None else [t]
        if case["out"] == "e4m3":
            top = torch.linalg.vector_norm(y, float("inf"), dim=-1)
            scale = torch.where(top > 0, top / E4M3_MAX, 1.0)
            return [y / scale[:, None], scale, *stream]
        outs, grads, leaves = [y, *stream], [s[n].double() for n in ("dy", "dstream") if s.get(n) is not None], [x, r, w]
    else:
        x, w = wide("x", "x_scale"), wide("w", "w_scale")
        z = torch.einsum("mk,nk->mn", x, w)
        if case["op"] == "gated":
            up = wide("up", "up_scale")
            y, leaves = _activation64(case["act"], z) * torch.einsum("mk,nk->mn", x, up), [x, w, up]
        else:
            b, r = wide("b"), wide("residual")
            y = _activation64(case["act"], z if b is None else z + b)
            y, leaves = (y if r is None else y + r), [x, w, b, r]
        outs, grads = [y], [s["dy"].double()] if case["train"] else []
    if not case["train"]:
        return outs
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, [x for x in leaves if x is not None], grads))
