"""Routing, dispatch / combine and the block norms in 64 bits, for the tests."""

import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def clean(logits):
    """NaN counts as minus infinity, plus infinity as the largest finite 32-bit value."""
    l = logits.double()
    return torch.where(l.isnan(), -math.inf, l.clamp(max=3.402823466e38))


def probabilities(l, scoring):
    if scoring == "sigmoid":
        return torch.sigmoid(l)
    top = l.amax(-1, keepdim=True)
    e = torch.where(l == -math.inf, 0.0, torch.exp(l - torch.where(top == -math.inf, 0.0, top)))
    return e / e.sum(-1, keepdim=True).clamp(min=1e-300)


def order(score):
    """Experts by falling score, lowest number first where equal."""
    return torch.sort(score, dim=-1, descending=True, stable=True).indices


def route(logits, top_k, bias=None, scoring="softmax", groups=1, top_groups=None, group_score="max", mask=None):
    """(idx, rows, offsets) of the choice."""
    l = clean(logits)
    t, e = l.shape
    s = l if bias is None else probabilities(l, scoring) + clean(bias)
    if bias is not None:
        s = torch.where((l == -math.inf) | (clean(bias) == -math.inf), -math.inf, s)
    top_groups = groups if top_groups is None else top_groups
    out = torch.zeros(t, e, dtype=torch.bool, device=l.device)
    if top_groups < groups:
        by = s
        if group_score == "top2" and bias is None:
            by = torch.where(l == -math.inf, -math.inf, probabilities(l, scoring))
        best = by.view(t, groups, e // groups).sort(-1, descending=True).values
        score = best[..., 0] + best[..., 1] if group_score == "top2" else best[..., 0]
        kept = order(score)[:, :top_groups]
        keep = torch.zeros(t, groups, dtype=torch.bool, device=l.device).scatter_(1, kept, True)
        out = ~keep.repeat_interleave(e // groups, 1)
    # Experts of groups that went stand behind those that are out by their logit: sort by two keys.
    idx = order(s)
    idx = idx.gather(1, torch.sort(out.gather(1, idx).int(), dim=-1, stable=True).indices)[:, :top_k]
    if mask is not None:
        idx = torch.where(mask[:, None], idx, -1)
    flat = torch.where(idx < 0, e, idx).flatten()
    rows = torch.empty_like(flat)
    rows[torch.sort(flat, stable=True).indices] = torch.arange(flat.numel(), device=l.device)
    offsets = torch.cat([flat.new_zeros(1), torch.bincount(flat, minlength=e + 1)[:e].cumsum(0)])
    return idx, torch.where(idx < 0, -1, rows.view(idx.shape)), offsets


def weights(logits, idx, scoring, renormalise, scale):
    """Weights of a given choice, differentiable in `logits` (float64)."""
    live = (idx >= 0) & (logits.gather(1, idx.clamp(min=0)) != -math.inf)
    if renormalise:
        l = torch.where(live, logits.gather(1, idx.clamp(min=0)), -1e300)
        if scoring == "softmax":
            q = torch.exp(l - l.amax(-1, keepdim=True).detach())
        else:
            q = torch.exp(torch.nn.functional.logsigmoid(l) - torch.nn.functional.logsigmoid(l).amax(-1, keepdim=True).detach())
        q = torch.where(live, q, 0.0)
        w = q / q.sum(-1, keepdim=True).clamp(min=1e-300)
    else:
        p = torch.sigmoid(logits) if scoring == "sigmoid" else torch.softmax(logits, -1)
        w = torch.where(live, p.gather(1, idx.clamp(min=0)), 0.0)
    return scale * w


def rms(z, gamma, eps):
    return z * torch.rsqrt((z * z).mean(-1, keepdim=True) + eps) * (1 if gamma is None else gamma)


def block_norm(residual, x, gamma, post_gamma, gate, scale, eps):
    """(y, h) with every argument in float64; gate [hidden] or [sequences, hidden]."""
    u = x if post_gamma is None else rms(x, post_gamma, eps)
    if gate is not None:
        g = gate.view(-1, 1, gate.shape[-1])
        u = (u.reshape(g.shape[0], -1, u.shape[-1]) * g).view(u.shape)
    h = scale * residual + u
    return (None if gamma is None else rms(h, gamma, eps)), h
