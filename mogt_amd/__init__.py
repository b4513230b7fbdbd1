"""MI355X-native (gfx950) MOGT scan operator.

Public surface:
  - ``mogt_amd.ops``: ``diag_scan``, ``coupled_rank_scan``, ``ssm_scan`` and
    ``short_conv`` with their single-token forms ``ssm_step`` and
    ``short_conv_step`` (torch.ops.mogt.*).
Native code lives in ``mogt_amd/csrc`` (HIP, C ABI declared in
``include/mogt_scan.h``) and is built in-tree into ``mogt_amd/lib``.
"""
from . import _lib, ops  # noqa: F401
from .ops import coupled_rank_scan, dense_scan, diag_scan  # noqa: F401
from .ops import short_conv, short_conv_step, ssm_scan, ssm_step  # noqa: F401

__all__ = ["diag_scan", "coupled_rank_scan", "ssm_scan", "ssm_step", "short_conv", "short_conv_step"]
