"""CPU checks of the norm and the products around a mixer: what the C ABI and the layers refuse (nothing is launched)."""

import pytest
import torch

from jax_linear_attention_b200 import _lib, layers

BF16, F16, F32, E4M3 = 0, 1, 2, 3
P = 4096  # an aligned address that is never followed: every call below is refused before its launch


def _text():
    return _lib.load().jla_last_error().decode()


def _linear(dtype=BF16, out_dtype=None, rows=4, depth=64, out=64, x=P, stride=None, w=P, xs=None, ws=None, bias=None, act=0,
            res=None, y=P):
    out_dtype = (BF16 if dtype == E4M3 else dtype) if out_dtype is None else out_dtype
    return _lib.load().jla_linear_fwd(dtype, out_dtype, rows, depth, out, x, depth if stride is None else stride, w, xs, ws,
                                      bias, act, res, y, None, None)


@pytest.mark.parametrize("change, text", [
    (dict(dtype=F32), "bf16, f16 or e4m3"), (dict(dtype=7), "bf16, f16 or e4m3"), (dict(out_dtype=F16), "operands' type"),
    (dict(out_dtype=F32), "output must be"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"),
    (dict(depth=60), "multiple of 8"), (dict(depth=0), "multiple of 8"), (dict(out=65), "of 8"), (dict(out=0), "of 8"),
    (dict(dtype=E4M3, depth=72, xs=P, ws=P), "multiple of 16"), (dict(dtype=E4M3), "scales"), (dict(xs=P), "scales"),
    (dict(dtype=E4M3, xs=P), "scales"), (dict(act=4), "activation"), (dict(act=-1), "activation"), (dict(stride=56), "rows of x"),
    (dict(stride=68), "rows of x"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(y=None), "null"),
    (dict(x=P + 8), "aligned"), (dict(w=P + 2), "aligned"), (dict(y=P + 4), "aligned"), (dict(bias=P + 4), "aligned"),
    (dict(res=P + 2), "aligned"),
])
def test_linear_abi_refuses(change, text):
    assert _linear(**change) == _lib.ERR_BAD_ARGUMENT
    assert text in _text()


def test_no_rows_is_no_launch():
    assert _linear(rows=0, x=None, y=None) == _lib.OK
    lib = _lib.load()
    assert lib.jla_gated_linear_fwd(BF16, BF16, 0, 64, 64, None, 64, None, None, None, None, None, 1, None, None, None, None) == 0
    assert lib.jla_linear_bwd_input(BF16, 0, 64, 64, None, None, None, None, None, None) == 0
    assert lib.jla_gated_activation_bwd(BF16, 0, 64, 1, None, None, None, None, None, None) == 0
    assert lib.jla_rms_norm_fwd(BF16, 0, 64, None, None, None, 1e-6, 0, None, None, None, None, None) == 0


def test_gradient_abi_refuses():
    lib = _lib.load()
    bad = _lib.ERR_BAD_ARGUMENT
    assert lib.jla_linear_bwd_input(F32, 4, 64, 64, P, P, None, None, P, None) == bad
    assert lib.jla_linear_bwd_input(BF16, 4, 64, 64, P, P, P, None, P, None) == bad  # half of a second pair
    assert lib.jla_linear_bwd_input(BF16, 4, 62, 64, P, P, None, None, P, None) == bad
    assert lib.jla_linear_bwd_weight(E4M3, 4, 64, 64, P, None, P, 64, P, None, None) == bad
    assert lib.jla_linear_bwd_weight(BF16, 4, 64, 64, P, P, P, 64, P, None, None) == bad
    assert lib.jla_linear_bwd_weight(BF16, 4, 64, 64, P, None, P, 60, P, None, None) == bad
    assert lib.jla_activation_bwd(BF16, 4, 64, 1, None, P, None, P, P, 1 << 20, None) == bad  # an activation needs z
    assert lib.jla_activation_bwd(BF16, 4, 60, 0, None, P, None, P, P, 1 << 20, None) == bad
    assert lib.jla_activation_bwd(BF16, 4, 64, 0, None, P, None, P, P, 16, None) == _lib.ERR_WORKSPACE
    assert lib.jla_gated_activation_bwd(F32, 4, 64, 1, P, P, P, P, P, None) == bad
    need = lib.jla_activation_bwd_scratch_bytes(4, 64)
    assert 64 * 4 <= need <= 592 * 64 * 4


@pytest.mark.parametrize("change, text", [
    (dict(dtype=E4M3), "dtype"), (dict(rows=-1), "rows"), (dict(dim=0), "width"), (dict(dim=16385), "width"),
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(res=P), "null"), (dict(e4m3=1), "null"),
])
def test_rms_norm_abi_refuses(change, text):
    a = dict(dtype=BF16, rows=4, dim=64, x=P, res=None, w=P, e4m3=0, y=P, stream=None, scale=None) | change
    rc = _lib.load().jla_rms_norm_fwd(a["dtype"], a["rows"], a["dim"], a["x"], a["res"], a["w"], 1e-6, a["e4m3"], a["y"],
                                      a["stream"], None, a["scale"], None)
    assert rc == _lib.ERR_BAD_ARGUMENT and text in _text()


def test_rms_norm_backward_abi_refuses():
    lib = _lib.load()
    need = lib.jla_rms_norm_bwd_scratch_bytes(100, 64)
    assert need >= 64 * 4
    assert lib.jla_rms_norm_bwd(F32, 100, 64, P, None, P, P, P, None, P, P, P, need - 1, None) == _lib.ERR_WORKSPACE
    assert lib.jla_rms_norm_bwd(F32, 100, 64, P, None, None, P, P, None, P, None, None, 0, None) == _lib.ERR_BAD_ARGUMENT
    assert lib.jla_rms_norm_bwd_scratch_bytes(0, 64) == 0 and lib.jla_rms_norm_bwd_scratch_bytes(5, 20000) == 0


def test_layers_have_no_cpu_fallback():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(64, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no CPU fallback"):
        layers.rms_norm(x, torch.ones(64))
    with pytest.raises(ValueError, match="no CPU fallback"):
        layers.linear(x, w)
    with pytest.raises(ValueError, match="no CPU fallback"):
        layers.gated_linear(x, w, w)
    with pytest.raises(ValueError, match="activation"):
        layers.linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="activation"):
        layers.gated_linear(x, w, w, activation=None)
