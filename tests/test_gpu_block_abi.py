"""Calls of the norm's C ABI that the layers do not make."""

import pytest
import torch

from jax_linear_attention_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows, dim", [(1, 64), (300, 2048), (7, 33)])
@pytest.mark.parametrize("dtype, code", [(torch.bfloat16, 0), (torch.float16, 1), (torch.float32, 2)])
def test_stream_without_a_residual(rows, dim, dtype, code):
    """The new stream of a sum with nothing is x; without a place for it, none is written."""
    x = torch.randn(rows, dim, device="cuda").to(dtype)
    w = torch.ones(dim, device="cuda")
    y, again = torch.empty_like(x), torch.empty_like(x)
    stream = torch.full_like(x, 9)
    _lib.launch("jla_rms_norm_fwd", x.device, code, rows, dim, x.data_ptr(), None, w.data_ptr(), 1e-6, 0, y.data_ptr(),
                stream.data_ptr(), None, None)
    _lib.launch("jla_rms_norm_fwd", x.device, code, rows, dim, x.data_ptr(), None, w.data_ptr(), 1e-6, 0, again.data_ptr(), None, None,
                None)
    assert bool((stream == x).all()) and bool((y == again).all())
