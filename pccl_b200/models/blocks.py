"""Model blocks that exercise the fused operators end to end.

``TensorParallelMLP``   Llama-style SwiGLU feed-forward under tensor + sequence parallelism:
    x[T/W, H] -(all-gather fused into the GEMM, SwiGLU in its epilogue)-> [T, F/W]
      -(GEMM with fused reduce-scatter)-> [T/W, H]: two kernels per block, no element-wise pass.
``MixtralMoEBlock``     residual + RMSNorm + expert-parallel top-2 MoE feed-forward.
``SparseMoEBlock``      a trainable MoE feed-forward on one GPU (replicate it and average its gradients with
    `pccl_b200.parallel.GradientBuckets`): any of `route_topk`'s routings, a norm behind the experts, a gate and a
    residual scale, built on `pccl_b200.ops.moe` and `pccl_b200.ops.norm`.

The inference blocks have a `reference()` in plain PyTorch (fp32) used by the tests.  The reference
framework has no model code; the shapes follow the Llama-3-8B / Mixtral-8x7B layers that its
benchmarks' collectives are sized for.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from ..ops.moe import combine, dispatch, route_topk
from ..ops.norm import residual_rms_norm
from ..ops.norm import rms_norm as _fused_rms_norm
from ..parallel.layers import ColumnParallelLinear, ExpertParallelMoE, RowParallelLinear


def rms_norm(x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * gamma.float()).to(x.dtype)


class TensorParallelMLP:
    def __init__(self, tokens: int, hidden: int, ffn_local: int, w_gate_up: torch.Tensor, w_down: torch.Tensor):
        """``w_gate_up [2 * ffn_local, hidden]`` (gate rows then up rows), ``w_down [hidden, ffn_local]``."""
        from ..ops.moe import interleave_gate_up
        self.tokens, self.hidden, self.ffn_local = tokens, hidden, ffn_local
        if ffn_local % 16:
            raise ValueError("ffn_local must be a multiple of 16")
        # Gate and up rows interleaved in groups of 16: one 32-column slice of the accumulator then
        # holds both halves of 16 outputs, which is what the fused epilogue combines.
        stacked = interleave_gate_up(w_gate_up[:ffn_local].unsqueeze(0), w_gate_up[ffn_local:].unsqueeze(0))
        self.up = ColumnParallelLinear(tokens, hidden, 2 * ffn_local, stacked, swiglu=True)
        self.down = RowParallelLinear(tokens, ffn_local, hidden, w_down)
        self.act = torch.empty(tokens, ffn_local, dtype=torch.bfloat16, device="cuda")

    def __call__(self, x_shard: torch.Tensor) -> torch.Tensor:
        self.up(x_shard, self.act)                                   # [T, F/W] = silu(gate) * up
        return self.down(self.act)                                   # [T/W, H]

    @staticmethod
    def reference(x_full: torch.Tensor, w_gate_up_all, w_down_all) -> torch.Tensor:
        """All ranks' weights (lists indexed by rank) applied to the gathered input, fp32."""
        out = torch.zeros(x_full.shape[0], w_down_all[0].shape[0], device=x_full.device)
        for wgu, wd in zip(w_gate_up_all, w_down_all):
            f = wgu.shape[0] // 2
            gu = x_full.float() @ wgu.float().t()
            act = (F.silu(gu[:, :f]) * gu[:, f:]).to(torch.bfloat16).float()
            out += act @ wd.float().t()
        return out


class MixtralMoEBlock:
    def __init__(self, tokens: int, hidden: int, ffn: int, experts: int, gamma: torch.Tensor, local: bool = False):
        self.gamma = gamma
        self.moe = ExpertParallelMoE(tokens, hidden, ffn, experts, local=local)

    def load(self, wg, w1, w3, w2) -> None:
        self.moe.load(wg, w1, w3, w2)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return x + self.moe(rms_norm(x, self.gamma))


class SparseMoEBlock(torch.nn.Module):
    """Norm, routed SwiGLU experts, norm behind, gate and residual, with gradients.

    ``forward(stream)`` returns ``(normed, stream)`` after the block: the new residual stream and, where
    ``next_gamma`` (the next block's ``gamma``) is given, that stream normed for the next block, which takes it as
    ``normed``.  ``routing`` holds the keyword arguments of `route_topk`; ``balance`` adds the float32 buffer
    ``bias``, which the caller moves to keep the experts' load even.  The experts' products are library matrix
    products over each expert's rows, so one host read of the row offsets stands in every forward pass.
    """

    def __init__(self, hidden: int, ffn: int, experts: int, top_k: int, *, post_norm: bool = False, gated: bool = False,
                 balance: bool = False, residual_scale: float = 1.0, eps: float = 1e-5,
                 dtype: torch.dtype = torch.bfloat16, device="cuda", **routing):
        super().__init__()

        def normal(*shape, scale):
            return torch.nn.Parameter((torch.randn(*shape, device=device) * scale).to(dtype))

        def ones():
            return torch.nn.Parameter(torch.ones(hidden, dtype=dtype, device=device))

        self.top_k, self.routing, self.residual_scale, self.eps = top_k, routing, residual_scale, eps
        self.gamma = ones()
        self.post_gamma = ones() if post_norm else None
        self.gate = ones() if gated else None
        self.register_buffer("bias", torch.zeros(experts, device=device) if balance else None)
        self.wg = normal(experts, hidden, scale=hidden ** -0.5)
        self.w13 = normal(experts, 2 * ffn, hidden, scale=hidden ** -0.5)
        self.w2 = normal(experts, hidden, ffn, scale=ffn ** -0.5)

    def experts(self, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        """Rows in expert order through their experts; unused rows become zero.

        Experts without rows are passed over, but for one where none has any: the weights get a gradient, of zero then,
        in every batch, so that ranks that average them always agree on what there is to reduce.
        """
        ends = offsets.tolist()
        parts = []
        for e in range(self.w2.shape[0]):
            if ends[e + 1] > ends[e] or (e == 0 and ends[-1] == 0):
                gate, up = (x[ends[e]:ends[e + 1]] @ self.w13[e].t()).chunk(2, dim=-1)
                parts.append((F.silu(gate) * up) @ self.w2[e].t())
        parts.append(x.new_zeros(x.shape[0] - ends[-1], x.shape[1]))
        return torch.cat(parts)

    def forward(self, stream: torch.Tensor, normed: torch.Tensor = None, next_gamma: torch.Tensor = None,
                mask: torch.Tensor = None):
        if normed is None:
            normed = _fused_rms_norm(stream, self.gamma, self.eps)
        logits = normed.float() @ self.wg.float().t()
        routing = route_topk(logits, self.top_k, bias=self.bias, mask=mask, **self.routing)
        out = combine(self.experts(dispatch(normed, routing), routing.offsets), routing)
        return residual_rms_norm(stream, out, next_gamma, post_gamma=self.post_gamma, gate=self.gate,
                                 residual_scale=self.residual_scale, eps=self.eps)
