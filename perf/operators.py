"""The operators around a block's matrix products, as they are timed: expert routing, the move of rows into
expert order and back, and the norms around a block with its gate and residual scale.

``own`` false: every operator in its plain form, elementary torch operations in 32 bits (the router's scores in
64, because the order of two near scores is part of the answer), rounded once at the end.  ``own`` true: the
calls a user makes of ``pccl_b200.ops``.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}

# Largest amounts of work of the listed cases, which drawn ones stay under: logits, values moved in 16 bits,
# values normed in 16 bits.
_MOST_LOGITS = 65536 * 256
_MOST_MOVED = 8192 * 4096 * 9
_MOST_NORMED = 16384 * 4096


# ---------------------------------------------------------------------------------------------------- the cases
def _route(name, tokens, experts, top_k, dtype, scoring, bias, groups, top_groups, group_score, renormalise, scale,
           live, train):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype,
            "scoring": scoring, "bias": bias, "groups": groups, "top_groups": top_groups, "group_score": group_score,
            "renormalise": renormalise, "scale": scale, "live": live, "train": train}


def _move(name, op, tokens, hidden, experts, top_k, dtype, live, train):
    return {"name": name, "op": op, "tokens": tokens, "hidden": hidden, "experts": experts, "top_k": top_k,
            "dtype": dtype, "live": live, "train": train}


def _norm(name, tokens, hidden, dtype, residual, pre, post, gates, scale, train):
    return {"name": name, "op": "norm", "tokens": tokens, "hidden": hidden, "dtype": dtype, "residual": residual,
            "pre": pre, "post": post, "gates": gates, "scale": scale, "train": train}


def listed():
    return [
        # One sequence being decoded: nothing but latency.
        _route("route, one token", 1, 64, 6, "bf16", "sigmoid", True, 8, 3, "top2", True, 2.5, 1.0, False),
        # A ragged batch of prompts padded to a fixed number of rows, softmax scores limited to the best groups.
        _route("route, padded prompts", 4001, 160, 6, "fp32", "softmax", False, 8, 3, "max", False, 16.0, 0.9, False),
        # A training step of the 8-expert layer that the MoE benchmark of this repository times.
        _route("route, training, 8 experts", 16384, 8, 2, "bf16", "softmax", False, 1, 1, "max", True, 1.0, 1.0, True),
        # A training step over many experts whose load a bias keeps even: the largest router.
        _route("route, training, 256 experts", 65536, 256, 8, "fp32", "sigmoid", True, 8, 4, "top2", True, 2.5, 1.0,
               True),
        # Rows into expert order: a batch of sequences being decoded, and a training step of the 8-expert layer.
        _move("dispatch, decoding", "dispatch", 32, 4096, 8, 2, "bf16", 1.0, False),
        _move("dispatch, training", "dispatch", 16384, 4096, 8, 2, "bf16", 1.0, True),
        # Rows back: padded prompts of odd width, and a training step with eight experts a token, the largest move.
        _move("combine, padded prompts", "combine", 1777, 1431, 64, 5, "fp16", 0.9, False),
        _move("combine, training", "combine", 8192, 4096, 64, 8, "bf16", 1.0, True),
        # The residual stream between two blocks while a few sequences are decoded.
        _norm("norm, decoding", 8, 4096, "bf16", "bf16", True, False, 0, 1.0, False),
        # Prompts of odd width through a block with a norm on both sides and one gate per channel.
        _norm("norm, prompts", 5001, 2055, "fp16", "fp16", True, True, 1, 1.0, False),
        # Training: eight sequences with a gate each, norms on both sides, a scaled residual: the largest norm.
        _norm("norm, training, gated", 16384, 4096, "bf16", "bf16", True, True, 8, 0.9, True),
        # Training with a residual stream held in 32 bits, the plain pre-norm block.
        _norm("norm, training, fp32 stream", 4100, 8192, "bf16", "fp32", True, False, 0, 1.0, True),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm, odd ones as often as even ones."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["route", "route", "dispatch", "combine", "norm", "norm"])
    train = rng.random() < 0.5
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    live = rng.choice([1.0, 1.0, 0.9])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        size = _spread(rng, 2, 512 // groups)
        experts = max(groups * size, 4)
        groups = groups if experts == groups * size else 1
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(10, top_groups * (experts // groups)))
        tokens = _spread(rng, 1, min(65536, _MOST_LOGITS // experts))
        scoring = rng.choice(["softmax", "sigmoid"])
        case = _route("", tokens, experts, top_k, rng.choice(["fp32", "fp32", "bf16", "fp16"]), scoring,
                      rng.random() < 0.5, groups, top_groups, rng.choice(["max", "top2"]) if experts // groups > 1 else "max",
                      rng.random() < 0.7, rng.choice([1.0, 2.5]), live, train)
    elif op == "norm":
        hidden = _spread(rng, 64, 16384)
        hidden = hidden // 64 * 64 if rng.random() < 0.6 else hidden
        residual = rng.choice([dtype, dtype, "fp32"])
        sequences = rng.choice([0, 0, 1, 2, 5])
        tokens = _spread(rng, 1, min(16384, _MOST_NORMED * 4 // (hidden * (_BYTES[dtype] + _BYTES[residual]))))
        tokens = max(1, tokens // max(1, sequences)) * max(1, sequences)
        pre = rng.random() < 0.85
        case = _norm("", tokens, hidden, dtype, residual, pre, rng.random() < 0.5, sequences, rng.choice([1.0, 0.9]),
                     train)
    else:
        hidden = _spread(rng, 64, 8192)
        hidden = hidden // 64 * 64 if rng.random() < 0.6 else hidden
        experts = rng.choice([8, 16, 60, 128])
        top_k = rng.randint(1, 8)
        tokens = _spread(rng, 1, min(16384, _MOST_MOVED * 2 // (hidden * (top_k + 1) * _BYTES[dtype])))
        case = _move("", op, tokens, hidden, experts, top_k, dtype, live, train)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    t, kind = case["tokens"], _TYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "norm":
        h = case["hidden"]
        state["x"] = normal(t, h).mul_(1.5).to(kind)
        state["residual"] = normal(t, h).mul_(2.0).to(_TYPES[case["residual"]])
        state["gamma"] = (1 + 0.1 * normal(h)).to(kind) if case["pre"] else None
        state["post_gamma"] = (1 + 0.1 * normal(h)).to(kind) if case["post"] else None
        gates = case["gates"]
        state["gate"] = (0.5 + 0.2 * normal(*((gates, h) if gates > 1 else (h,)))).to(kind) if gates else None
        if case["train"]:
            state["dy"] = normal(t, h).to(kind) if case["pre"] else None
            state["dh"] = normal(t, h).to(_TYPES[case["residual"]])
            for name in ("x", "residual", "gamma", "post_gamma", "gate"):
                if state[name] is not None:
                    state[name].requires_grad_(True)
        return state
    mask = torch.rand(t, device="cuda", generator=g) < case["live"] if case["live"] < 1 else None
    e, k = case["experts"], case["top_k"]
    if case["op"] == "route":
        state["logits"] = normal(t, e).mul_(1.5).to(kind).requires_grad_(case["train"])
        state["bias"] = 0.1 * normal(e) if case["bias"] else None
        state["mask"] = mask
        state["dweights"] = normal(t, k) if case["train"] else None
        return state
    # The routing that an earlier call has left in hand: distinct experts a token, and their rows in expert order.
    scores = torch.rand(t, e, device="cuda", generator=g)
    idx = scores.argsort(-1)[:, :k].to(torch.int32)
    weights = torch.softmax(normal(t, k), -1)
    if mask is not None:
        idx = torch.where(mask[:, None], idx, -1)
        weights = torch.where(mask[:, None], weights, 0.0)
    rows, offsets = _expert_order(idx, e)
    state.update(idx=idx, weights=weights.requires_grad_(case["train"] and case["op"] == "combine"), rows=rows,
                 offsets=offsets)
    h = case["hidden"]
    tall, wide = (t, t * k) if case["op"] == "dispatch" else (t * k, t)
    state["x"] = normal(tall, h).to(kind).requires_grad_(case["train"])
    state["dout"] = normal(wide, h).to(kind) if case["train"] else None
    return state


# ----------------------------------------------------------------------------------------------- the plain forms
def _expert_order(idx, experts):
    """Row of every choice when the choices are ordered by expert, tokens in order within one; -1 stays out."""
    flat = torch.where(idx < 0, experts, idx).flatten().long()
    order = torch.sort(flat, stable=True).indices
    rows = torch.empty_like(flat)
    rows[order] = torch.arange(flat.numel(), device=flat.device)
    counts = torch.bincount(flat, minlength=experts + 1)[:experts]
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=flat.device)
    offsets[1:] = counts.cumsum(0)
    return torch.where(idx < 0, -1, rows.view(idx.shape)).to(torch.int32), offsets


def _plain_scores(case, logits):
    l64 = logits.double()
    if case["scoring"] == "sigmoid":
        return 1 / (1 + torch.exp(-l64))
    top = torch.exp(l64 - l64.amax(-1, keepdim=True))
    return top / top.sum(-1, keepdim=True)


def _plain_route(s):
    case, logits = s["case"], s["logits"].detach()
    t, e = logits.shape
    k, groups = case["top_k"], case["groups"]
    p = _plain_scores(case, logits)
    by = p + s["bias"].double() if s["bias"] is not None else p
    if groups > 1 and case["top_groups"] < groups:
        split = by.view(t, groups, e // groups)
        if case["group_score"] == "top2":
            score = split.sort(-1, descending=True).values[..., :2].sum(-1)
        else:
            score = split.amax(-1)
        kept = score.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros(t, groups, dtype=torch.bool, device=logits.device)
        keep[torch.arange(t, device=logits.device)[:, None], kept] = True
        by = torch.where(keep.repeat_interleave(e // groups, 1), by, -math.inf)
    idx = by.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    chosen = p.gather(1, idx)
    total = chosen.sum(-1, keepdim=True)
    w = case["scale"] * (chosen / total if case["renormalise"] else chosen)
    out = {}
    if case["train"]:
        g = s["dweights"].double()
        if case["renormalise"]:
            g = (case["scale"] * g - (g * w).sum(-1, keepdim=True)) / total
        else:
            g = case["scale"] * g
        dp = torch.zeros_like(p)
        if s["mask"] is not None:
            g = torch.where(s["mask"][:, None], g, 0.0)
        dp.scatter_(1, idx, g)
        if case["scoring"] == "sigmoid":
            dl = dp * p * (1 - p)
        else:
            dl = p * (dp - (dp * p).sum(-1, keepdim=True))
        out["dlogits"] = dl.to(logits.dtype)
    if s["mask"] is not None:
        idx = torch.where(s["mask"][:, None], idx, -1)
        w = torch.where(s["mask"][:, None], w, 0.0)
    rows, offsets = _expert_order(idx, e)
    out.update(idx=idx.to(torch.int32), weights=w.float(), rows=rows, offsets=offsets)
    return out


def _plain_move(s):
    case, x, rows = s["case"], s["x"].detach(), s["rows"].long()
    t, k = rows.shape
    live = rows >= 0
    if case["op"] == "dispatch":
        out = torch.zeros(t * k, x.shape[1], dtype=x.dtype, device=x.device)
        token = torch.arange(t, device=x.device)[:, None].expand(t, k)
        out[rows[live]] = x[token[live]]
        if not case["train"]:
            return {"out": out}
        dout = s["dout"].float()[rows.clamp(min=0)]
        return {"out": out, "dx": torch.where(live[..., None], dout, 0.0).sum(1).to(x.dtype)}
    w = torch.where(live, s["weights"].detach(), 0.0)
    rows0 = rows.clamp(min=0)
    y = x.float()[rows0]
    out = (w[..., None] * y).sum(1).to(x.dtype)
    if not case["train"]:
        return {"out": out}
    dout = s["dout"].float()
    dx = torch.zeros(x.shape, dtype=torch.float32, device=x.device)
    scaled = w[..., None] * dout[:, None]
    dx[rows[live]] = scaled[live]
    dw = torch.where(live, (y * dout[:, None]).sum(-1), 0.0)
    return {"out": out, "dx": dx.to(x.dtype), "dweights": dw}


def _plain_norm(s):
    case = s["case"]
    t, hidden = s["x"].shape
    x, residual = s["x"].detach().float(), s["residual"].detach().float()
    gates = max(1, case["gates"])

    def rows_of(gate):
        return gate.detach().float().view(gates, 1, hidden).expand(gates, t // gates, hidden).reshape(t, hidden)

    eps = 1e-5
    out = {}
    u = x
    if case["post"]:
        r1 = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
        n1 = x * r1
        u = n1 * s["post_gamma"].detach().float()
    v = u * rows_of(s["gate"]) if case["gates"] else u
    h = case["scale"] * residual + v
    out["h"] = h.to(s["residual"].dtype)
    if case["pre"]:
        r2 = torch.rsqrt((h * h).mean(-1, keepdim=True) + eps)
        n2 = h * r2
        gamma = s["gamma"].detach().float()
        out["y"] = (n2 * gamma).to(s["x"].dtype)
    if not case["train"]:
        return out
    d = s["dh"].float()
    if case["pre"]:
        dy = s["dy"].float()
        a = dy * gamma
        d = d + r2 * (a - n2 * (a * n2).mean(-1, keepdim=True))
        out["dgamma"] = (dy * n2).sum(0).to(s["gamma"].dtype)
    out["dresidual"] = (case["scale"] * d).to(s["residual"].dtype)
    if case["gates"]:
        out["dgate"] = (d * u).view(gates, t // gates, hidden).sum(1).view(s["gate"].shape).to(s["gate"].dtype)
        d = d * rows_of(s["gate"])
    if case["post"]:
        out["dpost_gamma"] = (d * n1).sum(0).to(s["post_gamma"].dtype)
        b = d * s["post_gamma"].detach().float()
        d = r1 * (b - n1 * (b * n1).mean(-1, keepdim=True))
    out["dx"] = d.to(s["x"].dtype)
    return out


# --------------------------------------------------------------------------------------------- the framework's
def _own_route(s):
    from pccl_b200.ops import moe
    case = s["case"]
    r = moe.route_topk(s["logits"], case["top_k"], bias=s["bias"], scoring=case["scoring"], groups=case["groups"],
                       top_groups=case["top_groups"], group_score=case["group_score"],
                       renormalise=case["renormalise"], scale=case["scale"], mask=s["mask"])
    out = {"idx": r.idx, "weights": r.weights, "rows": r.rows, "offsets": r.offsets}
    if case["train"]:
        out["dlogits"], = torch.autograd.grad(r.weights, s["logits"], s["dweights"])
    return out


def _own_move(s):
    from pccl_b200.ops import moe
    case = s["case"]
    routing = moe.Routing(s["idx"], s["weights"], s["rows"], s["offsets"])
    if case["op"] == "dispatch":
        out = moe.dispatch(s["x"], routing)
        if not case["train"]:
            return {"out": out}
        return {"out": out, "dx": torch.autograd.grad(out, s["x"], s["dout"])[0]}
    out = moe.combine(s["x"], routing)
    if not case["train"]:
        return {"out": out}
    dx, dw = torch.autograd.grad(out, (s["x"], s["weights"]), s["dout"])
    return {"out": out, "dx": dx, "dweights": dw}


def _own_norm(s):
    from pccl_b200.ops import norm
    case = s["case"]
    y, h = norm.residual_rms_norm(s["residual"], s["x"], s["gamma"], post_gamma=s["post_gamma"], gate=s["gate"],
                                  residual_scale=case["scale"], eps=1e-5)
    out = {"h": h}
    if case["pre"]:
        out["y"] = y
    if not case["train"]:
        return out
    names = [n for n in ("x", "residual", "gamma", "post_gamma", "gate") if s[n] is not None]
    ends = ((y, h), (s["dy"], s["dh"])) if case["pre"] else ((h,), (s["dh"],))
    grads = torch.autograd.grad(ends[0], [s[n] for n in names], ends[1])
    out.update(zip(["d" + n for n in names], grads))
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_route(state) if op == "route" else _own_norm(state) if op == "norm" else _own_move(state)
    return _plain_route(state) if op == "route" else _plain_norm(state) if op == "norm" else _plain_move(state)


# ------------------------------------------------------------------------------------------- the least it can do
def work(case):
    """Bytes: each input read once and each output written once.  Operations: those of the formulas."""
    t, size, train = case["tokens"], _BYTES[case["dtype"]], case["train"]
    if case["op"] == "route":
        e, k = case["experts"], case["top_k"]
        moved = t * e * size + t * k * 12 + 4 * (e + 1) + (4 * e if case["bias"] else 0) + (t if case["live"] < 1 else 0)
        if train:
            moved += t * e * size + t * k * 4
        return {"bytes": moved, "flops": t * (6 * e + 8 * k) * (2 if train else 1)}
    h = case["hidden"]
    if case["op"] == "norm":
        rsize = _BYTES[case["residual"]]
        weights = h * size * (int(case["pre"]) + int(case["post"]) + case["gates"])
        moved = t * h * (size + 2 * rsize + (size if case["pre"] else 0)) + weights
        flops = t * h * (2 + 4 * int(case["pre"]) + 4 * int(case["post"]) + int(case["gates"] > 0))
        if train:
            moved += t * h * ((size if case["pre"] else 0) + rsize + size + rsize) + weights
            flops *= 3
        return {"bytes": moved, "flops": flops}
    k = case["top_k"]
    moved = t * h * size * (k + 1) + 4 * t * k * (2 if case["op"] == "combine" else 1)
    flops = 2 * t * k * h if case["op"] == "combine" else 0
    if train and case["op"] == "dispatch":
        moved += t * h * size * (k + 1)
        flops += t * k * h
    elif train:
        moved += t * h * size * (k + 1) + 4 * t * k
        flops += 3 * t * k * h
    return {"bytes": moved, "flops": flops}


# -------------------------------------------------------------------------------------------- from the definition
def _exact_route(s):
    case = s["case"]
    logits = s["logits"].detach().double().requires_grad_(True)
    t, e = logits.shape
    p = torch.sigmoid(logits) if case["scoring"] == "sigmoid" else torch.softmax(logits, -1)
    by = p.detach().clone()
    if s["bias"] is not None:
        by += s["bias"].double()
    number = torch.arange(e, device=by.device)
    size = e // case["groups"]

    def lowest_best(score):
        """Column of each row's largest value, the lowest where several hold it."""
        n = score.shape[1]
        at = torch.arange(n, device=score.device)
        return torch.where(score == score.amax(1, keepdim=True), at, n).amin(1)

    if case["top_groups"] < case["groups"]:
        columns = []
        for j in range(case["groups"]):
            part = by[:, j * size:(j + 1) * size]
            best = part.gather(1, lowest_best(part)[:, None])
            if case["group_score"] == "top2":
                rest = part.scatter(1, lowest_best(part)[:, None], -math.inf)
                best = best + rest.amax(1, keepdim=True)
            columns.append(best)
        left = torch.cat(columns, 1)
        taken = torch.zeros(t, e, dtype=torch.bool, device=by.device)
        for _ in range(case["top_groups"]):
            best = lowest_best(left)
            taken |= (number // size)[None] == best[:, None]
            left.scatter_(1, best[:, None], -math.inf)
        by[~taken] = -math.inf
    picks = []
    for _ in range(case["top_k"]):
        best = lowest_best(by)
        picks.append(best)
        by.scatter_(1, best[:, None], -math.inf)
    chosen = p.gather(1, torch.stack(picks, 1))
    w = chosen / chosen.sum(1, keepdim=True) if case["renormalise"] else chosen
    w = w * case["scale"]
    if s["mask"] is not None:
        w = w * s["mask"][:, None]
    out = {"idx": None, "weights": w.detach(), "rows": None, "offsets": None}
    if case["train"]:
        out["dlogits"], = torch.autograd.grad(w, logits, s["dweights"].double())
    return out


def _exact_move(s):
    case = s["case"]
    x = s["x"].detach().double().requires_grad_(True)
    weights = s["weights"].detach().double().requires_grad_(True)
    t, k = s["rows"].shape
    if case["op"] == "dispatch":
        # As a list of source tokens by row, the rest of the rows from a row of zeros behind the last token.
        source = torch.full((t * k + 1,), t, dtype=torch.long, device=x.device)
        rows = s["rows"].long().flatten()
        source[torch.where(rows < 0, t * k, rows)] = torch.arange(t * k, device=x.device) // k
        out = torch.cat([x, x.new_zeros(1, x.shape[1])])[source[:-1]]
    else:
        # Padding reads a row of zeros behind the last one.
        padded = torch.cat([x, x.new_zeros(1, x.shape[1])])
        out = 0
        for j in range(k):
            rows = s["rows"][:, j].long()
            out = out + weights[:, j, None] * padded[torch.where(rows < 0, t * k, rows)]
    if not case["train"]:
        return {"out": out.detach()}
    if case["op"] == "dispatch":
        return {"out": out.detach(), "dx": torch.autograd.grad(out, x, s["dout"].double())[0]}
    dx, dw = torch.autograd.grad(out, (x, weights), s["dout"].double())
    return {"out": out.detach(), "dx": dx, "dweights": dw}


def _exact_norm(s):
    case = s["case"]
    names = [n for n in ("x", "residual", "gamma", "post_gamma", "gate") if s[n] is not None]
    v = {n: s[n].detach().double().requires_grad_(True) for n in names}

    def norm(z, gamma):
        return gamma * z / (z.square().mean(-1, keepdim=True) + 1e-5).sqrt()

    u = norm(v["x"], v["post_gamma"]) if case["post"] else v["x"]
    if case["gates"]:
        t, hidden = u.shape
        u = (u.view(case["gates"], t // case["gates"], hidden) * v["gate"].view(case["gates"], 1, hidden)).view(t, hidden)
    h = v["residual"] * case["scale"] + u
    out = {"h": h}
    if case["pre"]:
        out["y"] = norm(h, v["gamma"])
    if case["train"]:
        ends = [h] + ([out["y"]] if case["pre"] else [])
        back = [s["dh"].double()] + ([s["dy"].double()] if case["pre"] else [])
        grads = torch.autograd.grad(ends, [v[n] for n in names], back)
        out.update(zip(["d" + n for n in names], grads))
    return {n: z.detach() for n, z in out.items()}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_route(s) if case["op"] == "route" else _exact_norm(s) if case["op"] == "norm" else _exact_move(s)
