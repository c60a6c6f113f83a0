"""mamba3_amd — MI355X-native (gfx950 HIP) Mamba-3 chunked-SSD forward path.

Drop-in for the public API of `mamba3` (mamba3/__init__.py:5-19): `import mamba3_amd as
mamba3` gives the same eight names.
"""

__version__ = "0.1.0"

from .layer import KulaMamba, RMSNorm
from .block import KulaMambaBlock, KulaMambaLM, SwiGLU
from .ssd import chunked_ssd, SSDOutput
from .scan import ssd_scan
# Operators beyond the reference's API, for training and for serving from 4-bit weights: attributes
# of the package, not among the eight names of `__all__`.
from .add_norm import add_rms_norm, add_rms_norm_mx
from .clip import clip_grad_norm_
from .loss import linear_cross_entropy
from .mlp import swiglu_mlp
from .mx import MXTensor, mx_linear, quantize_mx, silu_mul_mx
from .sample import sample_tokens

__all__ = [
    "KulaMamba",
    "KulaMambaBlock",
    "KulaMambaLM",
    "RMSNorm",
    "SwiGLU",
    "SSDOutput",
    "chunked_ssd",
    "ssd_scan",
]
