"""ksmm_amd: Kronecker-sparse matrix multiplication for MI355X (gfx950).

``KSLinear(patterns, weights, algo='kernel', dtype, bs_last)`` keeps the reference's API;
``algo='kernel'`` runs hand-written HIP kernels through the C ABI of libksmm_hip.so.
"""
from .layer import (KSLinear, bmm_bs_first, bmm_bs_last, from_abcd_to_dense,  # noqa: F401
                    from_bmm_format_to_dense, from_kernel_format_to_dense, generate_factor,
                    quantize_fp8)
from .kernel import Kernel, query_tile  # noqa: F401
from .block import (GatedKernel, KSFeedForward, KSGatedLinear, NormKernel, ResidualNorm, gated_linear,  # noqa: F401
                    pack_gated, residual_norm)
from .muon import KSMuon, muon_update, orthogonalize  # noqa: F401
from .mx import (KSFeedForwardMX, KSGatedLinearMX, KSLinearMX, MXFactor, MXKernel, MXLinear, MXTensor, mx_linear,  # noqa: F401
                 pack_block, pack_mx, quantize_mx)
from .adamw import KSAdamW, adamw_moments, adamw_update  # noqa: F401
