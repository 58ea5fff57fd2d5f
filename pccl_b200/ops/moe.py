"""Expert-parallel Mixture-of-Experts feed-forward (top-2 routing, SwiGLU experts).

Three kernels per call, all on the caller's stream:

1. route + dispatch: router logits, softmax top-2 with renormalised gates, and each token row
   pushed straight into the receive buffer of the rank that owns its expert (NVLink stores);
2. expert GEMM 1 on the tcgen05 tensor cores over the filled rows only, SwiGLU in the epilogue;
3. expert GEMM 2 whose epilogue multiplies by the gate and stores each row into the combine
   buffer of the token's home rank, followed in the same kernel by the two-way sum per token.

Experts are spread evenly over the ranks (``experts % world == 0``); a region of ``cap`` rows
per (local expert, source rank) is reserved so that no token is ever dropped.  Without a
process group (one GPU) an ordinary CUDA buffer stands in for the symmetric heap.
Construction is collective.  The reference has no MoE operator; the workload is its
all-to-all template's target use (pccl/dsl/algorithms/ring.py, build_alltoall).

For layers that route otherwise, or that are trained, the steps around the experts' products are operators of
their own, on ordinary tensors of one GPU and with gradients:

``route_topk``   scores (softmax or sigmoid, a bias for balance, groups), top-k, weights, expert order;
``dispatch``     token rows into expert order, one copy per choice;
``combine``      the experts' rows back to their tokens, weighted and summed.

They run on the tensors' device and its current stream, may be captured into a CUDA graph (a backward pass, as for any
torch operator, only while no eager graph of the same leaves is alive), and raise ``ValueError`` for arguments they do
not take.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import engine as _engine
from .tensor_parallel import _fence

_BLOCK = 128


def interleave_gate_up(w1: torch.Tensor, w3: torch.Tensor) -> torch.Tensor:
    """Stack ``w1`` (gate) and ``w3`` (up), each ``[experts, ffn, hidden]``, as the kernel reads them.

    Per expert, rows alternate in groups of 16: 16 gate rows, then the 16 up rows of the same
    hidden units, so one 32-column slice of the accumulator holds both halves of SwiGLU.
    Returns ``[experts * 2 * ffn, hidden]``.
    """
    e, f, h = w1.shape
    if f % 16:
        raise ValueError("ffn must be a multiple of 16")
    g = w1.reshape(e, f // 16, 1, 16, h)
    u = w3.reshape(e, f // 16, 1, 16, h)
    return torch.cat([g, u], dim=2).reshape(e * 2 * f, h).contiguous()


def moe_reference(x, wg, w1, w3, w2):
    """Plain fp32 PyTorch statement of the layer (all experts local), for tests."""
    xf = x.float()
    logits = xf @ wg.float().t()
    top, idx = logits.topk(2, dim=-1)
    gates = torch.softmax(top, dim=-1)
    out = torch.zeros_like(xf)
    for e in range(wg.shape[0]):
        for k in range(2):
            rows = (idx[:, k] == e).nonzero().squeeze(-1)
            if rows.numel() == 0:
                continue
            xe = xf[rows]
            h = torch.nn.functional.silu(xe @ w1[e].float().t()) * (xe @ w3[e].float().t())
            out[rows] += gates[rows, k, None] * (h.to(torch.bfloat16).float() @ w2[e].float().t())
    return out, idx, gates


def _round_up(v: int, m: int) -> int:
    return (v + m - 1) // m * m


class FusedMoE:
    """``out[tokens, hidden] = sum_k gate_k * expert_k(x)`` over the two routed experts of each token."""

    def __init__(self, tokens: int, hidden: int, ffn: int, experts: int, group=None, local: bool = False):
        self.tokens, self.hidden, self.ffn, self.experts = tokens, hidden, ffn, experts
        self.native = _engine.load_native().fused
        self.local = local
        if local:
            self.world, self.rank = 1, 0
        else:
            self.engine = _engine.get_engine()
            self.world, self.rank = self.engine.world, self.engine.rank
        if experts % self.world:
            raise ValueError(f"{experts} experts do not divide over {self.world} ranks")
        self.local_experts = experts // self.world
        self.cap = _round_up(tokens, _BLOCK)
        regions = self.local_experts * self.world
        sizes = [
            regions * self.cap * hidden * 2,        # recv
            regions * self.cap * 8,                 # meta
            _round_up(regions * 4, 256),            # counts
            256,                                    # ready flags
            256,                                    # done flags
            tokens * 2 * hidden * 2,                # combine
        ]
        if local:
            offsets, total = [], 0
            for s in sizes:
                offsets.append(total)
                total += _round_up(s, 256)
            self.heap = torch.zeros(total, dtype=torch.uint8, device="cuda")
            self.offsets = offsets
        else:
            self.heap = None
            self._buffers = [self.engine.empty_symmetric((_round_up(s, 256),), torch.uint8) for s in sizes]
            for b in self._buffers[2:5]:
                b.zero_()
            self.offsets = [b.heap_offset for b in self._buffers]
        self.h = torch.empty(regions * self.cap, ffn, dtype=torch.bfloat16, device="cuda")
        self.scratch = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
        self.cta_counter = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.topk_idx = torch.empty(tokens, 2, dtype=torch.int32, device="cuda")
        self.topk_gate = torch.empty(tokens, 2, dtype=torch.float32, device="cuda")
        self.epoch = 0
        self.wg = self.w13 = self.w2 = None
        if not local:
            _fence(group)

    def set_weights(self, wg: torch.Tensor, w1: torch.Tensor, w3: torch.Tensor, w2: torch.Tensor) -> None:
        """``wg [experts, hidden]`` (replicated); ``w1, w3 [local_experts, ffn, hidden]`` and
        ``w2 [local_experts, hidden, ffn]`` are this rank's experts."""
        le = self.local_experts
        if tuple(w1.shape) != (le, self.ffn, self.hidden) or tuple(w2.shape) != (le, self.hidden, self.ffn):
            raise ValueError("expert weights have the wrong shape")
        self.wg = wg.to(torch.bfloat16).contiguous()
        self.w13 = interleave_gate_up(w1.to(torch.bfloat16), w3.to(torch.bfloat16))
        self.w2 = w2.to(torch.bfloat16).reshape(le * self.hidden, self.ffn).contiguous()

    def __call__(self, x: torch.Tensor, out: torch.Tensor = None, ctas: int = 0, phases: int = 7) -> torch.Tensor:
        if self.wg is None:
            raise RuntimeError("set_weights() first")
        if tuple(x.shape) != (self.tokens, self.hidden) or x.dtype != torch.bfloat16:
            raise ValueError(f"x must be bf16 [{self.tokens}, {self.hidden}]")
        if out is None:
            out = torch.empty(self.tokens, self.hidden, dtype=torch.bfloat16, device=x.device)
        self.epoch += 1
        self.native.moe_forward(x.contiguous(), self.wg, self.w13, self.w2, self.h, out, self.scratch,
                                self.cta_counter, self.offsets, self.cap, self.epoch, self.heap, ctas, phases,
                                self.topk_idx, self.topk_gate)
        return out


def route(x: torch.Tensor, wg: torch.Tensor):
    """Router alone: ``(topk_idx [T,2] int32, gates [T,2] fp32, slots [T,2] int32, counts [E] int32)``."""
    native = _engine.load_native().fused
    tokens, experts = x.shape[0], wg.shape[0]
    scratch = torch.empty(experts + 1, dtype=torch.int32, device=x.device)
    idx = torch.empty(tokens, 2, dtype=torch.int32, device=x.device)
    gate = torch.empty(tokens, 2, dtype=torch.float32, device=x.device)
    slot = torch.empty(tokens, 2, dtype=torch.int32, device=x.device)
    counts = torch.empty(experts, dtype=torch.int32, device=x.device)
    native.moe_route(x.contiguous(), wg.contiguous(), scratch, idx, gate, slot, counts)
    return idx, gate, slot, counts


class Routing(NamedTuple):
    """What ``route_topk`` chose.  Rows ``offsets[e]`` to ``offsets[e + 1]`` of a batch in expert order belong to
    expert ``e``, tokens in order; rows from ``offsets[-1]`` on are unused (there are some only with a mask).

    A caller may leave choices out (experts of bounded capacity, say): ``routing._replace(rows=...)`` with -1, or any
    number outside the batch, in their places.  No two choices may name the same row: which of them it then holds, or
    takes its gradient from, is not defined."""

    idx: torch.Tensor       # [tokens, top_k] int32, best first; -1 for masked tokens
    weights: torch.Tensor   # [tokens, top_k] float32, differentiable
    rows: torch.Tensor      # [tokens, top_k] int32: row of each choice in expert order; -1 for masked tokens
    offsets: torch.Tensor   # [experts + 1] int32

    def __reduce__(self):
        # Parts of one allocation cannot be written to a file together where their types differ, and each would bring
        # all of it along.
        return type(self), tuple(t.clone() for t in self)


_block = None


def _block_native():
    global _block
    if _block is None:
        _block = _engine.load_native().block
    return _block


def route_topk(logits: torch.Tensor, top_k: int, *, bias: Optional[torch.Tensor] = None, scoring: str = "softmax",
               groups: int = 1, top_groups: Optional[int] = None, group_score: str = "max", renormalise: bool = True,
               scale: float = 1.0, mask: Optional[torch.Tensor] = None) -> Routing:
    """Choose ``top_k`` experts per token from router logits ``[tokens, experts]`` (float32, float16, bfloat16).

    ``p = softmax(logits)`` or ``sigmoid(logits)`` (``scoring``).  Experts are ranked by ``s = p + bias`` (``bias``
    float32 ``[experts]``, for an even load; it changes the choice alone and has no gradient).  With ``groups``
    equal groups of neighbouring experts only those of the ``top_groups`` best stay, a group counting by its best
    score (``group_score="max"``) or the sum of its two best (``"top2"``).  Ties go to the lowest number; scores
    are told apart to 64 bits (without a bias by the logits themselves).  The weights are
    ``scale * p / sum(p over the choice)``, or ``scale * p`` with ``renormalise=False``.

    A logit of minus infinity or NaN takes an expert out: its score is minus infinity whatever its bias, it is
    chosen only where nothing else is left, and then with weight 0.  Plus infinity counts as the largest finite
    logit.  Tokens where ``mask`` (bool ``[tokens]``) is false choose nothing: index and row -1, weight 0.

    Up to 1024 experts, 32 groups, 31 choices, and ``tokens * top_k`` below 2^31 - 2^16.  ``weights`` carries the gradient
    of ``logits`` (once: it cannot be differentiated twice, and there is no forward mode); the order of the choices within
    an expert is that of the tokens, on every run.  The four results are parts of one allocation, which holds the
    workspace too and lives as long as any of them.  Save the `Routing` itself, or clones of its parts: a part alone
    would bring the whole allocation along, and torch refuses ``idx`` and ``weights`` of one in the same file.
    """
    if scoring not in ("softmax", "sigmoid"):
        raise ValueError(f"route_topk: scoring must be 'softmax' or 'sigmoid', not {scoring!r}")
    if group_score not in ("max", "top2"):
        raise ValueError(f"route_topk: group_score must be 'max' or 'top2', not {group_score!r}")
    return Routing(*_block_native().route_topk(logits, top_k, bias, scoring == "sigmoid", groups,
                                               groups if top_groups is None else top_groups, group_score == "top2",
                                               renormalise, scale, mask))


def dispatch(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """``out[routing.rows[t, k]] = x[t]``: ``[tokens * top_k, hidden]`` in expert order, for the experts' products.

    Rows that no choice names become zero: those from ``routing.offsets[-1]`` on, and those of choices that were left
    out.  The gradient of ``x`` sums its copies in 32 bits.  ``x`` is float32, float16 or bfloat16 ``[tokens, hidden]``,
    rows at any distance.
    """
    return _block_native().dispatch(x, routing.rows, routing.offsets)


def combine(y: torch.Tensor, routing: Routing) -> torch.Tensor:
    """``out[t] = sum_k routing.weights[t, k] * y[routing.rows[t, k]]``: the experts' rows back to their tokens.

    The sum is taken in 32 bits in the order of the choices and rounded once; a token without choices gets zeros.
    Gradients go to ``y`` (zero in rows that no choice names) and to ``routing.weights``.
    """
    return _block_native().combine(y, routing.weights, routing.rows, routing.offsets)
