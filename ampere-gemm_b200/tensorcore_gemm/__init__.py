"""B200-native drop-in for the reference ``tensorcore_gemm`` package.

Public surface identical to the reference (tensorcore_gemm/__init__.py:1-3).
Importing the package also registers ``torch.ops.tensorcore_gemm.mm`` (the
same GEMM as a dispatcher operator with autograd, see ``ops``) and the
operators of the modules ``norm`` (layer norm), ``ffn`` (gated feed-forward
block) and ``logprobs`` (token log probabilities).
"""
from . import ffn as _ffn  # noqa: F401  (registers torch.ops.tensorcore_gemm.gated_ffn)
from . import logprobs as _logprobs  # noqa: F401  (registers torch.ops.tensorcore_gemm.token_logprobs)
from . import norm as _norm  # noqa: F401  (registers torch.ops.tensorcore_gemm.layer_norm)
from . import ops as _ops  # noqa: F401  (registers torch.ops.tensorcore_gemm.mm)
from .gemm import KERNEL_MODES, gemm, gemm_pretransposed, is_supported

__all__ = ["KERNEL_MODES", "gemm", "gemm_pretransposed", "is_supported"]
