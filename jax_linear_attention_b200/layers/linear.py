"""The matrix products of a block with what follows them in their epilogue: ``linear`` for the projections in front of and
behind a mixer (bias, activation, the residual's addition), ``gated_linear`` for the first half of a gated feed-forward
block (both projections, the activation and the product in one kernel). The reference leaves these to XLA's fusions and to
``src/jla/ops/mosaic_gpu/fused_gemm.py``.

A whole block is ``rms_norm`` -> ``linear`` -> the mixer -> ``linear`` with the residual, then ``rms_norm`` ->
``gated_linear`` -> ``linear`` with the residual. Operands are bf16 or f16 (with gradients), or e4m3 with one float32 scale a
row of ``x`` and a row of the weight (serving; ``rms_norm`` leaves its output in that form). Products are summed in float32
by the tensor cores, and everything up to the rounding of the result is float32.

Forward is one launch, of a kernel for many tokens or of one for few (``csrc/product_tc.cu``, ``csrc/few_tokens.cu``).
Backward, ``dx`` and ``dW`` are one launch each (both halves of a gated block together), after one for the activation's
gradient and the bias's where there are any. Before an activation the product is kept in float32 for the backward pass.
"""

from __future__ import annotations

import torch

from .. import _lib
from ..ops.cuda import aligned, nothing_to_differentiate

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float8_e4m3fn: 3}
_ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "sigmoid": 3}
_E4M3 = torch.float8_e4m3fn


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(x, width: int):
    """``x [..., width]`` as ``(matrix, elements between its rows)`` without a copy where its rows allow 16-byte loads."""
    try:
        x = x.view(-1, width)
    except RuntimeError:
        x = x.reshape(-1, width)
    if x.shape[0] <= 1 and x.stride(1) == 1:
        stride = width
    else:
        stride = x.stride(0)
    if x.stride(1) != 1 or stride < width or stride * x.element_size() % 16 or x.data_ptr() % 16:
        x, stride = aligned(x), width
    return x, stride


def _empty(rows, cols, dtype, device):
    return torch.empty(rows, cols, dtype=dtype, device=device)


def _activation_code(name: str, activation, allowed) -> int:
    if activation not in allowed:
        raise ValueError(f"{name}: unsupported activation {activation!r}; expected one of {allowed}")
    return _ACTIVATIONS[activation]


def _check(name: str, x, weights, scales, x_scale, out_dtype):
    """Checks the operands; returns the output's dtype."""
    for label, t in (("x", x), *((f"weight {i}", w) for i, w in enumerate(weights))):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"{name}: {label} must be a CUDA tensor: the 'cuda' implementation has no CPU fallback")
    w = weights[0]
    if x.dtype not in _DTYPES or any(t.dtype != x.dtype for t in weights):
        raise ValueError(f"{name}: x and the weights must share one of {sorted(str(d) for d in _DTYPES)}; got {x.dtype}, "
                         f"{[str(t.dtype) for t in weights]}")
    if w.ndim != 2 or x.ndim < 1 or x.shape[-1] != w.shape[1] or any(t.shape != w.shape for t in weights):
        raise ValueError(f"{name}: expected x [..., in] and weights [out, in]; got {tuple(x.shape)}, "
                         f"{[tuple(t.shape) for t in weights]}")
    if any(t.device != x.device for t in weights):
        raise ValueError(f"{name}: the weights must be on {x.device}")
    out, depth = w.shape
    step = 16 if x.dtype == _E4M3 else 8
    if depth < step or depth % step or out < 8 or out % 8:
        raise ValueError(f"{name}: in features must be a multiple of {step} and out features of 8; got {depth} and {out}")
    if x.dtype != _E4M3:
        if x_scale is not None or any(s is not None for s in scales):
            raise ValueError(f"{name}: scales go with e4m3 operands only")
        if out_dtype not in (None, x.dtype):
            raise ValueError(f"{name}: out_dtype must be {x.dtype}; got {out_dtype}")
        return x.dtype
    for label, s, shape in (("x_scale", x_scale, x.shape[:-1]), *(("weight scale", s, (out,)) for s in scales)):
        if s is None or s.dtype != torch.float32 or s.shape != shape or s.device != x.device:
            raise ValueError(f"{name}: e4m3 operands need a float32 {label} {tuple(shape)} on {x.device}")
    if out_dtype not in (None, torch.bfloat16, torch.float16):
        raise ValueError(f"{name}: out_dtype must be torch.bfloat16 or torch.float16; got {out_dtype}")
    return out_dtype or torch.bfloat16


def _linear_fwd(x, stride, weight, x_scale, weight_scale, bias, residual, act: int, out_dtype, keep_z: bool):
    rows, depth = x.shape
    out = weight.shape[0]
    y = _empty(rows, out, out_dtype, x.device)
    z = _empty(rows, out, torch.float32, x.device) if keep_z else None
    _lib.launch("jla_linear_fwd", x.device, _DTYPES[x.dtype], _DTYPES[out_dtype], rows, depth, out, x.data_ptr(), stride,
                weight.data_ptr(), _ptr(x_scale), _ptr(weight_scale), _ptr(bias), act, _ptr(residual), y.data_ptr(), _ptr(z))
    return y, z


def _grad_input(dz, weight, dz2=None, weight2=None):
    rows, out = dz.shape
    dx = _empty(rows, weight.shape[1], dz.dtype, dz.device)
    _lib.launch("jla_linear_bwd_input", dz.device, _DTYPES[dz.dtype], rows, weight.shape[1], out, dz.data_ptr(),
                weight.data_ptr(), _ptr(dz2), _ptr(weight2), dx.data_ptr())
    return dx


def _grad_weight(dz, x, stride, dz2=None):
    rows, out = dz.shape
    depth = x.shape[1]
    dw = _empty(out, depth, dz.dtype, dz.device)
    dw2 = None if dz2 is None else torch.empty_like(dw)
    _lib.launch("jla_linear_bwd_weight", dz.device, _DTYPES[dz.dtype], rows, depth, out, dz.data_ptr(), _ptr(dz2),
                x.data_ptr(), stride, dw.data_ptr(), _ptr(dw2))
    return dw, dw2


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act: int):
        rows, stride = _rows(x, weight.shape[1])
        out_shape = (*x.shape[:-1], weight.shape[0])
        y, z = _linear_fwd(rows, stride, weight, None, None, bias, aligned(residual), act, x.dtype, act != 0)
        ctx.save_for_backward(rows, weight, z)
        ctx.act, ctx.stride, ctx.x_shape = act, stride, x.shape
        return y.view(out_shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        rows, out = x.shape[0], weight.shape[0]
        flat = aligned(dy.reshape(rows, out))
        dz, db = flat, None
        if (z is not None and (need_x or need_w)) or need_b:
            dz = flat if z is None else torch.empty_like(flat)
            scratch = None
            if need_b:
                db = torch.empty(out, dtype=torch.float32, device=x.device)
                scratch = torch.empty(_lib.load().jla_activation_bwd_scratch_bytes(rows, out), dtype=torch.uint8, device=x.device)
            _lib.launch("jla_activation_bwd", x.device, _DTYPES[x.dtype], rows, out, ctx.act, _ptr(z), flat.data_ptr(),
                        None if z is None else dz.data_ptr(), _ptr(db), _ptr(scratch), 0 if scratch is None else scratch.numel())
        dx = _grad_input(dz, weight).view(ctx.x_shape) if need_x else None
        dw = _grad_weight(dz, x, ctx.stride)[0] if need_w else None
        return dx, dw, db, dy if need_r else None, None


def linear(x, weight, bias=None, *, activation: str | None = None, residual=None, x_scale=None, weight_scale=None,
           out_dtype=None):
    """``act(x @ weight.T + bias) + residual``, in one launch.

    ``x [..., in]`` and ``weight [out, in]`` in bf16 or f16 (``in`` and ``out`` multiples of 8), ``bias [out]``, ``residual
    [..., out]`` in the output's dtype; ``activation`` is None, ``"silu"``, ``"gelu"`` (tanh form) or ``"sigmoid"``. The rows of
    ``x`` may lie apart (a slice of a wider tensor). Gradients of ``x``, ``weight``, ``bias`` and ``residual``.

    e4m3 operands (``in`` a multiple of 16) take ``x_scale [...]`` and ``weight_scale [out]`` in float32: the product is that
    of ``x * x_scale[..., None]`` and ``weight * weight_scale[:, None]``; the output is bf16, or f16 with ``out_dtype``. This
    form has no gradient and is refused where one would be recorded.
    """
    act = _activation_code("linear", activation, (None, "silu", "gelu", "sigmoid"))
    dtype = _check("linear", x, (weight,), (weight_scale,), x_scale, out_dtype)
    out_shape = (*x.shape[:-1], weight.shape[0])
    if bias is not None and (bias.shape != weight.shape[:1] or bias.device != x.device):
        raise ValueError(f"linear: bias must be [{weight.shape[0]}] on {x.device}; got {tuple(bias.shape)} on {bias.device}")
    if residual is not None and (residual.shape != out_shape or residual.dtype != dtype or residual.device != x.device):
        raise ValueError(f"linear: residual must be {dtype} {out_shape} on {x.device}; got {residual.dtype} "
                         f"{tuple(residual.shape)} on {residual.device}")
    plain = nothing_to_differentiate((x, weight, bias, residual, x_scale, weight_scale))
    if x.dtype == _E4M3 and not plain:
        raise ValueError("linear: e4m3 operands have no gradient: call it under torch.no_grad()")
    weight = aligned(weight)
    bias = None if bias is None else aligned(bias.float())
    if not plain:
        return _Linear.apply(x, weight, bias, residual, act)
    rows, stride = _rows(x, weight.shape[1])
    y, _ = _linear_fwd(rows, stride, weight, aligned(x_scale), aligned(weight_scale), bias, aligned(residual), act, dtype, False)
    return y.view(out_shape)


def _gated_fwd(x, stride, w_gate, w_up, x_scale, gate_scale, up_scale, act: int, out_dtype, keep: bool):
    rows, depth = x.shape
    out = w_gate.shape[0]
    h = _empty(rows, out, out_dtype, x.device)
    g, u = (_empty(rows, out, torch.float32, x.device) for _ in range(2)) if keep else (None, None)
    _lib.launch("jla_gated_linear_fwd", x.device, _DTYPES[x.dtype], _DTYPES[out_dtype], rows, depth, out, x.data_ptr(), stride,
                w_gate.data_ptr(), w_up.data_ptr(), _ptr(x_scale), _ptr(gate_scale), _ptr(up_scale), act, h.data_ptr(),
                _ptr(g), _ptr(u))
    return h, g, u


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act: int):
        rows, stride = _rows(x, w_gate.shape[1])
        h, g, u = _gated_fwd(rows, stride, w_gate, w_up, None, None, None, act, x.dtype, True)
        ctx.save_for_backward(rows, w_gate, w_up, g, u)
        ctx.act, ctx.stride, ctx.x_shape = act, stride, x.shape
        return h.view(*x.shape[:-1], w_gate.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, g, u = ctx.saved_tensors
        need_x, need_g, need_u, _ = ctx.needs_input_grad
        rows, out = g.shape
        dh = aligned(dh.reshape(rows, out))
        dg, du = torch.empty_like(dh), torch.empty_like(dh)
        _lib.launch("jla_gated_activation_bwd", x.device, _DTYPES[x.dtype], rows, out, ctx.act, g.data_ptr(), u.data_ptr(),
                    dh.data_ptr(), dg.data_ptr(), du.data_ptr())
        dx = _grad_input(dg, w_gate, du, w_up).view(ctx.x_shape) if need_x else None
        d_gate = d_up = None
        if need_g and need_u:
            d_gate, d_up = _grad_weight(dg, x, ctx.stride, du)
        elif need_g:
            d_gate = _grad_weight(dg, x, ctx.stride)[0]
        elif need_u:
            d_up = _grad_weight(du, x, ctx.stride)[0]
        return dx, d_gate, d_up, None


def gated_linear(x, w_gate, w_up, *, activation: str = "silu", x_scale=None, gate_scale=None, up_scale=None, out_dtype=None):
    """``act(x @ w_gate.T) * (x @ w_up.T)``, both products, the activation and their product in one launch.

    ``x [..., in]``, ``w_gate`` and ``w_up [out, in]`` in bf16 or f16 (``in`` and ``out`` multiples of 8); ``activation`` is
    ``"silu"``, ``"gelu"`` (tanh form) or ``"sigmoid"``. Gradients of ``x`` and both weights. e4m3 operands take ``x_scale
    [...]``, ``gate_scale [out]`` and ``up_scale [out]`` as in ``linear``, without gradients.
    """
    act = _activation_code("gated_linear", activation, ("silu", "gelu", "sigmoid"))
    dtype = _check("gated_linear", x, (w_gate, w_up), (gate_scale, up_scale), x_scale, out_dtype)
    plain = nothing_to_differentiate((x, w_gate, w_up, x_scale, gate_scale, up_scale))
    if x.dtype == _E4M3 and not plain:
        raise ValueError("gated_linear: e4m3 operands have no gradient: call it under torch.no_grad()")
    w_gate, w_up = aligned(w_gate), aligned(w_up)
    if not plain:
        return _GatedLinear.apply(x, w_gate, w_up, act)
    rows, stride = _rows(x, w_gate.shape[1])
    h, _, _ = _gated_fwd(rows, stride, w_gate, w_up, aligned(x_scale), aligned(gate_scale), aligned(up_scale), act, dtype, False)
    return h.view(*x.shape[:-1], w_gate.shape[0])
