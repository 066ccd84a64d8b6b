"""The matrix products of a block with what follows them in their epilogue: ``linear`` for the projections in front of and
behind a mixer (bias, activation, the residual's addition), ``gated_linear`` for the first half of a gated feed-forward
block (both projections, the activation and the product in one kernel). The reference leaves these to XLA's fusions and to
``src/jla/ops/mosaic_gpu/fused_gemm.py``.

A whole block is ``rms_norm`` -> ``linear`` -> the mixer -> ``linear`` with the residual, then ``rms_norm`` ->
``gated_linear`` -> ``linear`` with the residual. Operands are bf16 or f16 (with gradients), or e4m3 with one float32 scale a
row of ``x`` and a row of the weight (serving; ``rms_norm`` leaves its output in that form). Products are summed in float32
by the tensor cores, and everything up to the rounding of the result is float32. float32 operands are not taken: the tensor
cores cut their sums off instead of rounding them (4e-6 of the result at a depth of 4096, 2e-5 at 16384 with random signs, 6.5e-5
where all terms are positive), which 16-bit results do not see and float32 ones would. Contractions of more than 16384 (e4m3:
32768) are summed in parts of that length, joined in float32 with rounding, so that this does not grow with the number of tokens
that the gradient of a weight sums over.

Forward is one launch, of a kernel for many tokens or of one for few (``csrc/product_tc.cu``, ``csrc/few_tokens.cu``).
Backward, ``dx`` and ``dW`` are one launch each (both halves of a gated block together), after one for the activation's
gradient and the bias's where there are any. Before an activation the product is kept in float32 for the backward pass; the
activation's gradient is rounded to the operands' type before the products (half a step more in ``dx`` and ``dW``). Only what the
wanted gradients read is kept.
A backward pass is captured into a graph like any other work, but not while an eager autograd graph of its leaves is alive on the
default stream, nor where a part of its graph was made there (a weight that was transposed before the capture): that raises.
"""

from __future__ import annotations

import torch

from .. import _lib

_DTYPES = (torch.bfloat16, torch.float16, torch.float8_e4m3fn)
_ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "sigmoid": 3}
_E4M3 = torch.float8_e4m3fn


def _code(name: str, activation, allowed) -> int:
    if activation not in allowed:
        raise ValueError(f"{name}: unsupported activation {activation!r}; expected one of {allowed}")
    return _ACTIVATIONS[activation]


def _no_tensor(name: str, **operands):
    for label, t in operands.items():
        if t is not None and not isinstance(t, torch.Tensor):
            raise ValueError(f"{name}: {label} must be a tensor or None; got {type(t).__name__}")


def _refuse(name: str, x, weights, scales, x_scale, out_dtype):
    """Says what keeps ``csrc/torch_ops.cpp`` from taking these operands; returns the output's dtype where nothing does."""
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
    if not (1 <= depth <= 1 << 24 and 1 <= out <= 1 << 24):
        raise ValueError(f"{name}: in and out features must be 1 .. 2^24; got {depth} and {out}")
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


def linear(x, weight, bias=None, *, activation: str | None = None, residual=None, x_scale=None, weight_scale=None,
           out_dtype=None):
    """``act(x @ weight.T + bias) + residual``, in one launch.

    ``x [..., in]`` and ``weight [out, in]`` in bf16 or f16, ``bias [out]``, ``residual [..., out]`` in the output's dtype;
    ``activation`` is None, ``"silu"``, ``"gelu"`` (tanh form) or ``"sigmoid"``. The rows of ``x`` may lie apart (a slice of a wider
    tensor). Gradients of ``x``, ``weight``, ``bias`` and ``residual``. ``in`` and ``out`` that are no multiples of 8 (``in`` of 16
    in e4m3) cost copies of the operands with zeros up to the next one: lay such weights out wider where that counts.

    e4m3 operands take ``x_scale [...]`` and ``weight_scale [out]`` in float32: the product is that
    of ``x * x_scale[..., None]`` and ``weight * weight_scale[:, None]``; the output is bf16, or f16 with ``out_dtype``. This
    form has no gradient and is refused where one would be recorded.
    """
    act = _code("linear", activation, (None, "silu", "gelu", "sigmoid"))
    y = (_lib._torch_ops or _lib.torch_ops()).linear(x, weight, bias, act, residual, x_scale, weight_scale, out_dtype)
    if y is not None:
        return y
    _no_tensor("linear", bias=bias, residual=residual, x_scale=x_scale, weight_scale=weight_scale)
    dtype = _refuse("linear", x, (weight,), (weight_scale,), x_scale, out_dtype)
    shape = (*x.shape[:-1], weight.shape[0])
    if bias is not None and (bias.shape != weight.shape[:1] or bias.device != x.device or not bias.is_floating_point()):
        raise ValueError(f"linear: bias must be floating [{weight.shape[0]}] on {x.device}; got {bias.dtype} {tuple(bias.shape)} on "
                         f"{bias.device}")
    if residual is not None and (residual.shape != shape or residual.dtype != dtype or residual.device != x.device):
        raise ValueError(f"linear: residual must be {dtype} {shape} on {x.device}; got {residual.dtype} "
                         f"{tuple(residual.shape)} on {residual.device}")
    raise ValueError("linear: e4m3 operands have no gradient: call it under torch.no_grad()")


def gated_linear(x, w_gate, w_up, *, activation: str = "silu", x_scale=None, gate_scale=None, up_scale=None, out_dtype=None):
    """``act(x @ w_gate.T) * (x @ w_up.T)``, both products, the activation and their product in one launch.

    ``x [..., in]``, ``w_gate`` and ``w_up [out, in]`` in bf16 or f16 (widths as in ``linear``); ``activation`` is ``"silu"``, ``"gelu"`` (tanh form) or ``"sigmoid"``. Gradients of ``x`` and both weights. e4m3 operands take ``x_scale
    [...]``, ``gate_scale [out]`` and ``up_scale [out]`` as in ``linear``, without gradients.
    """
    act = _code("gated_linear", activation, ("silu", "gelu", "sigmoid"))
    h = (_lib._torch_ops or _lib.torch_ops()).gated_linear(x, w_gate, w_up, act, x_scale, gate_scale, up_scale, out_dtype)
    if h is not None:
        return h
    _no_tensor("gated_linear", x_scale=x_scale, gate_scale=gate_scale, up_scale=up_scale)
    _refuse("gated_linear", x, (w_gate, w_up), (gate_scale, up_scale), x_scale, out_dtype)
    raise ValueError("gated_linear: e4m3 operands have no gradient: call it under torch.no_grad()")
