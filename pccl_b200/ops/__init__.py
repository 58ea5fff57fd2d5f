"""Fused compute + collective operators built on hand-written tcgen05 kernels, and the operators around a
block's products: expert routing, dispatch and combine (`moe`) and the norms around a block (`norm`)."""

from . import gemm, moe, norm
from .moe import FusedMoE, Routing, combine, dispatch, route_topk
from .norm import residual_rms_norm, rms_norm
from .tensor_parallel import AllGatherGemm, AllReduceResidualRMSNorm, GemmReduceScatter

__all__ = ["gemm", "moe", "FusedMoE", "GemmReduceScatter", "AllGatherGemm", "AllReduceResidualRMSNorm",
           "Routing", "route_topk", "dispatch", "combine", "norm", "rms_norm", "residual_rms_norm"]
