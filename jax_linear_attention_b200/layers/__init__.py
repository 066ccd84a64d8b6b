"""Callers of the hot path that the reference keeps in ``jla.layers``: the Mamba-2 SSD mapping, the q / k prologue
(short convolution + SiLU + L2 norm), the gate activations of the Gated DeltaNet / KDA mixers and their gated output
norm; and what stands around a mixer in a block: the residual stream's RMS norm, the projections and the gated
feed-forward block."""
from .conv import short_conv  # noqa: F401
from .gates import gate_prologue  # noqa: F401
from .norm import gated_rms_norm, rms_norm  # noqa: F401
from .products import gated_linear, linear  # noqa: F401
from .ssm import mamba2_ssd  # noqa: F401
