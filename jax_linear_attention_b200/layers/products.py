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
    """``x [..., width]`` as ``(tensor, rows, elements between rows)``, without a copy where its rows allow 16-byte loads."""
    if not x.is_contiguous():
        try:
            flat = x.view(-1, width)
        except RuntimeError:
            flat = x.contiguous()
        else:
            stride = flat.stride(0)
            if flat.stride(1) == 1 and stride >= width and not (stride * x.element_size() | x.data_ptr()) & 15:
                return flat, flat.shape[0], stride
        x = flat
    return aligned(x), x.numel() // width, width


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


def _plainly_fine(x, weight, out_dtype) -> bool:
    """Whether a call without scales has nothing that ``_check`` would object to (a decoding step spends a fifth of its host
    time there)."""
    dtype, shape = x.dtype, weight.shape
    return ((dtype is torch.bfloat16 or dtype is torch.float16) and weight.dtype is dtype and len(shape) == 2 and x.is_cuda
            and x.get_device() == weight.get_device() and x.ndim > 0 and x.shape[-1] == shape[1] and shape[0] > 0
            and shape[1] > 0 and not (shape[0] | shape[1]) & 7 and (out_dtype is None or out_dtype is dtype))


def _linear_fwd(x, rows, stride, shape, weight, x_scale, weight_scale, bias, residual, act: int, out_dtype, keep_z: bool):
    device, (out, depth) = x.device, weight.shape
    y = torch.empty(shape, dtype=out_dtype, device=device)
    z = torch.empty(rows, out, dtype=torch.float32, device=device) if keep_z else None
    _lib.launch("jla_linear_fwd", device, _DTYPES[x.dtype], _DTYPES[out_dtype], rows, depth, out, x.data_ptr(), stride,
                weight.data_ptr(), _ptr(x_scale), _ptr(weight_scale), _ptr(bias), act, _ptr(residual), y.data_ptr(), _ptr(z))
    return y, z


def _grad_input(shape, dz, weight, dz2=None, weight2=None):
    out, depth = weight.shape
    dx = torch.empty(shape, dtype=weight.dtype, device=weight.device)
    _lib.launch("jla_linear_bwd_input", weight.device, _DTYPES[weight.dtype], dx.numel() // depth, depth, out, dz.data_ptr(),
                weight.data_ptr(), _ptr(dz2), _ptr(weight2), dx.data_ptr())
    return dx


def _grad_weight(weight, dz, x, rows, stride, dz2=None):
    out, depth = weight.shape
    dw = torch.empty_like(weight)
    dw2 = None if dz2 is None else torch.empty_like(weight)
    _lib.launch("jla_linear_bwd_weight", weight.device, _DTYPES[weight.dtype], rows, depth, out, dz.data_ptr(), _ptr(dz2),
                x.data_ptr(), stride, dw.data_ptr(), _ptr(dw2))
    return dw, dw2


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act: int, shape):
        flat, rows, stride = _rows(x, weight.shape[1])
        y, z = _linear_fwd(flat, rows, stride, shape, weight, None, None, bias, aligned(residual), act, x.dtype, act != 0)
        ctx.save_for_backward(flat, weight, z)
        ctx.cfg = act, rows, stride, x.shape
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        act, rows, stride, x_shape = ctx.cfg
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        flat = aligned(dy)
        dz, db = flat, None
        if need_b or (z is not None and (need_x or need_w)):
            out, device = weight.shape[0], weight.device
            dz = flat if z is None else torch.empty_like(flat)
            scratch, nbytes = None, 0
            if need_b:
                nbytes = _lib.load().jla_activation_bwd_scratch_bytes(rows, out)
                db = torch.empty(out, dtype=torch.float32, device=device)
                scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
            _lib.launch("jla_activation_bwd", device, _DTYPES[weight.dtype], rows, out, act, _ptr(z), flat.data_ptr(),
                        None if z is None else dz.data_ptr(), _ptr(db), _ptr(scratch), nbytes)
        dx = _grad_input(x_shape, dz, weight) if need_x else None
        dw = _grad_weight(weight, dz, x, rows, stride)[0] if need_w else None
        return dx, dw, db, dy if need_r else None, None, None


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
    if x_scale is None and weight_scale is None and _plainly_fine(x, weight, out_dtype):
        dtype = x.dtype
    else:
        dtype = _check("linear", x, (weight,), (weight_scale,), x_scale, out_dtype)
    shape = (*x.shape[:-1], weight.shape[0])
    if bias is not None:
        if bias.shape != weight.shape[:1] or bias.device != x.device:
            raise ValueError(f"linear: bias must be [{weight.shape[0]}] on {x.device}; got {tuple(bias.shape)} on {bias.device}")
        bias = aligned(bias if bias.dtype is torch.float32 else bias.float())
    if residual is not None and (residual.shape != shape or residual.dtype is not dtype or residual.device != x.device):
        raise ValueError(f"linear: residual must be {dtype} {shape} on {x.device}; got {residual.dtype} "
                         f"{tuple(residual.shape)} on {residual.device}")
    plain = nothing_to_differentiate((x, weight, bias, residual, x_scale, weight_scale))
    weight = aligned(weight)
    if plain:
        flat, rows, stride = _rows(x, weight.shape[1])
        return _linear_fwd(flat, rows, stride, shape, weight, aligned(x_scale), aligned(weight_scale), bias, aligned(residual),
                           act, dtype, False)[0]
    if x.dtype is _E4M3:
        raise ValueError("linear: e4m3 operands have no gradient: call it under torch.no_grad()")
    return _Linear.apply(x, weight, bias, residual, act, shape)


def _gated_fwd(x, rows, stride, shape, w_gate, w_up, x_scale, gate_scale, up_scale, act: int, out_dtype, keep: bool):
    device, (out, depth) = x.device, w_gate.shape
    h = torch.empty(shape, dtype=out_dtype, device=device)
    g, u = (torch.empty(rows, out, dtype=torch.float32, device=device) for _ in range(2)) if keep else (None, None)
    _lib.launch("jla_gated_linear_fwd", device, _DTYPES[x.dtype], _DTYPES[out_dtype], rows, depth, out, x.data_ptr(), stride,
                w_gate.data_ptr(), w_up.data_ptr(), _ptr(x_scale), _ptr(gate_scale), _ptr(up_scale), act, h.data_ptr(),
                _ptr(g), _ptr(u))
    return h, g, u


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act: int, shape):
        flat, rows, stride = _rows(x, w_gate.shape[1])
        h, g, u = _gated_fwd(flat, rows, stride, shape, w_gate, w_up, None, None, None, act, x.dtype, True)
        ctx.save_for_backward(flat, w_gate, w_up, g, u)
        ctx.cfg = act, rows, stride, x.shape
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, g, u = ctx.saved_tensors
        act, rows, stride, x_shape = ctx.cfg
        need_x, need_g, need_u = ctx.needs_input_grad[:3]
        dh = aligned(dh)
        dg, du = torch.empty_like(dh), torch.empty_like(dh)
        _lib.launch("jla_gated_activation_bwd", dh.device, _DTYPES[dh.dtype], rows, w_gate.shape[0], act, g.data_ptr(),
                    u.data_ptr(), dh.data_ptr(), dg.data_ptr(), du.data_ptr())
        dx = _grad_input(x_shape, dg, w_gate, du, w_up) if need_x else None
        d_gate = d_up = None
        if need_g and need_u:
            d_gate, d_up = _grad_weight(w_gate, dg, x, rows, stride, du)
        elif need_g:
            d_gate = _grad_weight(w_gate, dg, x, rows, stride)[0]
        elif need_u:
            d_up = _grad_weight(w_up, du, x, rows, stride)[0]
        return dx, d_gate, d_up, None, None


def gated_linear(x, w_gate, w_up, *, activation: str = "silu", x_scale=None, gate_scale=None, up_scale=None, out_dtype=None):
    """``act(x @ w_gate.T) * (x @ w_up.T)``, both products, the activation and their product in one launch.

    ``x [..., in]``, ``w_gate`` and ``w_up [out, in]`` in bf16 or f16 (``in`` and ``out`` multiples of 8); ``activation`` is
    ``"silu"``, ``"gelu"`` (tanh form) or ``"sigmoid"``. Gradients of ``x`` and both weights. e4m3 operands take ``x_scale
    [...]``, ``gate_scale [out]`` and ``up_scale [out]`` as in ``linear``, without gradients.
    """
    act = _activation_code("gated_linear", activation, ("silu", "gelu", "sigmoid"))
    if (x_scale is None and gate_scale is None and up_scale is None and _plainly_fine(x, w_gate, out_dtype)
            and w_up.dtype is x.dtype and w_up.shape == w_gate.shape and w_up.device == x.device):
        dtype = x.dtype
    else:
        dtype = _check("gated_linear", x, (w_gate, w_up), (gate_scale, up_scale), x_scale, out_dtype)
    shape = (*x.shape[:-1], w_gate.shape[0])
    plain = nothing_to_differentiate((x, w_gate, w_up, x_scale, gate_scale, up_scale))
    w_gate, w_up = aligned(w_gate), aligned(w_up)
    if plain:
        flat, rows, stride = _rows(x, w_gate.shape[1])
        return _gated_fwd(flat, rows, stride, shape, w_gate, w_up, aligned(x_scale), aligned(gate_scale), aligned(up_scale), act,
                          dtype, False)[0]
    if x.dtype is _E4M3:
        raise ValueError("gated_linear: e4m3 operands have no gradient: call it under torch.no_grad()")
    return _GatedLinear.apply(x, w_gate, w_up, act, shape)
