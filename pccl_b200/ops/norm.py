"""Norms around a block, fused with the block's gate and the residual's scale (one kernel, with gradients).

``rms_norm``            ``y = x / sqrt(mean(x^2) + eps) * gamma``
``residual_rms_norm``   what stands between two blocks of a residual stream, in one pass over its rows:
                        the norm behind a block, its gate, the residual sum and the norm before the next block.

They run on the tensors' device and its current stream, may be captured into a CUDA graph (a backward pass, as for any
torch operator, only while no eager graph of the same leaves is alive), and raise ``ValueError`` for arguments they do
not take.  ``pccl_b200.ops.AllReduceResidualRMSNorm`` is the form for partial outputs that are first summed over ranks.
The reference has no norm operator.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import engine as _engine

_block = None


def _block_native():
    global _block
    if _block is None:
        _block = _engine.load_native().block
    return _block


def rms_norm(x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """``x [..., hidden]`` (float32, float16, bfloat16; hidden up to 16384) normed and scaled by ``gamma [hidden]``,
    which has the type of ``x`` or float32.  Differentiable once."""
    return _block_native().residual_rms_norm(x, None, gamma, None, None, 1.0, eps)[0]


def residual_rms_norm(residual: torch.Tensor, x: torch.Tensor, gamma: Optional[torch.Tensor] = None, *,
                      post_gamma: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                      residual_scale: float = 1.0, eps: float = 1e-5
                      ) -> Tuple[Optional[torch.Tensor], torch.Tensor]:
    """``(y, h)`` of ``h = residual_scale * residual + gate * norm(x) * post_gamma`` and ``y = norm(h) * gamma``.

    ``x`` is a block's output and ``residual`` the stream it joins, both ``[..., hidden]`` (hidden up to 16384);
    ``norm(z) = z / sqrt(mean(z^2) + eps)`` over the last dimension.  Without ``post_gamma`` the block's output is
    not normed, without ``gate`` not gated, and without ``gamma`` there is no norm before the next block and ``y``
    is None.  ``gate`` is ``[hidden]``, or ``[sequences, hidden]`` for as many equal runs of consecutive rows.

    ``x`` is float32, float16 or bfloat16; ``residual`` and ``h`` have its type or float32, ``y`` has its type, and
    each weight has its type or float32.  Everything is computed in 32 bits and rounded once; ``y`` is formed from
    ``h`` before that is rounded.  Gradients (once) go to every tensor; the weights' are summed in a fixed order.
    """
    if x is None:
        raise ValueError("residual_rms_norm: x is the block's output; for a norm alone use rms_norm")
    return _block_native().residual_rms_norm(residual, x, gamma, post_gamma, gate, residual_scale, eps)
