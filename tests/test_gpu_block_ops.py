"""Expert routing, dispatch / combine and the block norms on the GPU against 64-bit statements of them.

Tolerances count roundings.  One 32-bit operation is off by 2^-24 of its result, CUDA's expf, division and rsqrtf
by at most 2^-22; a result rounded to its type by HALF_STEP of its value (TINY near zero).  Sums of n terms are off
by n 2^-24 of the sum of the terms' sizes.
"""

import math

import pytest
import torch

import block_reference as ref
from block_reference import HALF_STEP, TINY
from pccl_b200.ops import Routing, combine, dispatch, residual_rms_norm, rms_norm, route_topk

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _close(got, want, slack, what=""):
    """|got - want| <= half a step of want's type + slack, elementwise."""
    bound = HALF_STEP[got.dtype] * want.abs() * (1 + 2 ** -10) + TINY[got.dtype] + slack
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off - bound)[bad].max())}" \
                                f" at {float(want[bad].abs().max())}"


# ------------------------------------------------------------------------------------------------- routing
def _check_route(logits, top_k, mask=None, bias=None, grad=True, **how):
    scoring, renormalise, scale = how.get("scoring", "softmax"), how.get("renormalise", True), how.get("scale", 1.0)
    logits = logits.detach().requires_grad_(grad)
    got = route_topk(logits, top_k, bias=bias, mask=mask, **how)
    idx, rows, offsets = ref.route(logits.detach(), top_k, bias, scoring, how.get("groups", 1), how.get("top_groups"),
                                   how.get("group_score", "max"), mask)
    assert got.idx.dtype == got.rows.dtype == got.offsets.dtype == torch.int32 and got.weights.dtype == torch.float32
    assert torch.equal(got.idx.long(), idx)
    assert torch.equal(got.rows.long(), rows)
    assert torch.equal(got.offsets.long(), offsets)
    # exp of arguments below 32 in size 2^-19 + 2^-22, sums of at most 31 + 5 (or 1024 / 32 + 5) terms 37 2^-24,
    # two quotients and the scale: below 2^-17 in all.
    l64 = ref.clean(logits.detach()).requires_grad_(True)
    want = ref.weights(l64, idx, scoring, renormalise, scale)
    torch.testing.assert_close(got.weights.double(), want.detach(), rtol=2 ** -17, atol=2 ** -126)
    if not grad:
        return got
    dw = _normal(_gen(5), *got.weights.shape)
    dl, = torch.autograd.grad(got.weights, logits, dw)
    dwant, = torch.autograd.grad(want, l64, dw.double())
    dwant = dwant.nan_to_num()
    # dl_e = c p_e (g_e - sum g p): each factor off by 2^-17 of the terms it is made of.
    share = ref.weights(l64.detach(), idx, scoring, renormalise, abs(scale))
    size = torch.zeros_like(dwant)
    if not renormalise and scoring == "softmax":
        size = abs(scale) * torch.softmax(l64.detach(), -1).nan_to_num() * (dw.double().abs() * share).sum(-1, keepdim=True)
    live = idx >= 0
    size.scatter_add_(1, idx.clamp(min=0), torch.where(live, share * (dw.double().abs() + (dw.double().abs() * share).sum(
        -1, keepdim=True) / max(abs(scale), 1e-30)), 0.0))
    assert dl.dtype == logits.dtype
    _close(dl, dwant, 2 ** -15 * size + 2 ** -126, "dlogits")
    return got


ROUTES = [
    # tokens, experts, top_k, how
    (1, 1, 1, dict()),
    (1, 64, 6, dict(scoring="sigmoid", groups=8, top_groups=3, group_score="top2", bias=True, scale=2.5)),
    (33, 8, 2, dict()),
    (257, 8, 8, dict(renormalise=False, scale=16.0)),
    (1000, 7, 3, dict(scoring="sigmoid", bias=True)),
    (700, 160, 6, dict(groups=8, top_groups=3, renormalise=False, scale=16.0)),
    (513, 96, 5, dict(groups=3, top_groups=2, group_score="top2", scoring="sigmoid")),
    (129, 100, 4, dict(groups=5, top_groups=2, bias=True)),
    (300, 256, 8, dict(scoring="sigmoid", groups=8, top_groups=4, group_score="top2", bias=True, scale=2.5)),
    (300, 384, 8, dict(scoring="sigmoid", renormalise=False, bias=True)),
    (70, 1024, 31, dict(bias=True)),
    (65, 1000, 31, dict(groups=20, top_groups=7, group_score="top2", scoring="sigmoid", renormalise=False)),
    (5000, 40, 4, dict(bias=True)),
    (20000, 32, 3, dict(groups=32, top_groups=5)),
    (64, 2, 1, dict(groups=2, top_groups=1)),
    # Around the sizes at which tokens go to more blocks, and lanes to more experts.
    (24, 9, 3, dict()), (25, 9, 3, dict(bias=True)), (148 * 8 + 1, 65, 9, dict()), (148 * 32 + 3, 33, 2, dict(scoring="sigmoid")),
    (1024, 8, 2, dict(bias=True)), (1025, 5, 5, dict(groups=5, top_groups=5)), (129, 31, 31, dict(renormalise=False)),
    (200, 192, 7, dict(groups=4, top_groups=3, bias=True)), (150, 192, 7, dict(groups=6, top_groups=3, group_score="top2")),
    (99, 510, 12, dict(groups=3, top_groups=2, bias=True, scoring="sigmoid")),
    (180, 8, 3, dict(groups=4, top_groups=2, group_score="top2", scoring="sigmoid", bias=True)),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", ROUTES, ids=lambda c: f"{c[0]}x{c[1]}k{c[2]}")
def test_route_topk(case, dtype):
    tokens, experts, top_k, how = case
    how = dict(how)
    g = _gen(tokens + experts)
    bias = 0.1 * _normal(g, experts) if how.pop("bias", False) else None
    logits = (1.5 * _normal(g, tokens, experts)).to(dtype)
    _check_route(logits, top_k, bias=bias, **how)
    mask = torch.rand(tokens, device="cuda", generator=g) < 0.7
    _check_route(logits, top_k, bias=bias, mask=mask, **how)


@pytest.mark.parametrize("experts,how", [(16, dict()), (256, dict(scoring="sigmoid", groups=8, top_groups=4, group_score="top2")),
                                         (64, dict(groups=4, top_groups=2))])
def test_route_ties_go_to_the_lowest(experts, how):
    """Few distinct values, equal and distinct biases: the order is decided by numbers alone."""
    g = _gen(3)
    logits = torch.randint(-2, 2, (700, experts), device="cuda", generator=g).float()
    logits[:50] = 0.0
    logits[50:100] = -0.0
    logits[100:150, ::2] = -0.0
    for bias in (None, torch.zeros(experts, device="cuda"), torch.arange(experts, device="cuda").remainder(3) * 0.25):
        _check_route(logits, min(8, experts), bias=bias, **how)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_tells_near_scores_apart(scoring):
    """Scores whose difference is far below one 32-bit step of the score: the bias undoes the logits' differences."""
    g = _gen(4)
    logits = (0.5 * _normal(g, 1, 64)).repeat(600, 1)
    p = ref.probabilities(logits[:1].double(), scoring)
    bias = (1 - p[0]).float()                                     # all scores equal but for the bias's own rounding
    got = _check_route(logits, 8, bias=bias, scoring=scoring)
    assert got.idx.unique().numel() == 8                          # the same choice for the same row
    _check_route(logits + 1e-6 * _normal(g, 600, 64), 8, bias=bias, scoring=scoring)
    _check_route(logits + 1e-6 * _normal(g, 600, 64), 8, bias=bias, scoring=scoring, groups=8, top_groups=3, group_score="top2")


@pytest.mark.parametrize("experts", [8, 40, 256])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_ranks_near_pairs_again(scoring, experts):
    """Pairs of scores a few units of the last place apart, at every place of the choice and just behind it."""
    g = _gen(14)
    tokens, k = 400, min(6, experts // 2)
    logits = _normal(g, 1, experts).repeat(tokens, 1)
    p = ref.probabilities(logits[:1].double(), scoring)[0]
    bias = 0.05 * _normal(g, experts)
    ranked = ref.order((p + bias.double())[None])[0]
    for i in range(0, k + 1, 2):                                      # choice i + 1 meets choice i, the last the runner-up
        a, b = ranked[i], ranked[i + 1]
        bias[b] = (p[a] + bias[a].double() - p[b]).float()
    logits += 2e-7 * _normal(g, tokens, experts)
    _check_route(logits, k, bias=bias, scoring=scoring)
    _check_route(logits, k, bias=bias, scoring=scoring, groups=4, top_groups=2, group_score="top2")
    near = _normal(g, tokens, experts)                               # and logits alone, some equal, some a unit apart
    near[:, 1::2] = near[:, ::2]
    near[::3, 1::2] = torch.nextafter(near[::3, ::2], torch.full((), 10.0, device="cuda"))
    _check_route(near, k, scoring=scoring)
    _check_route(near, k, scoring=scoring, groups=4, top_groups=2)


@pytest.mark.parametrize("experts", [8, 24, 40, 64, 200, 256, 500])
@pytest.mark.parametrize("biased", [False, True])
def test_route_ranks_a_few_near_ones_among_many(experts, biased):
    """Two to seven experts a row within eight units of the last place, some equal, around the end of the choice; the
    rest far below."""
    g = _gen(15)
    tokens = 3000
    logits = _normal(g, tokens, experts) - 8
    few = torch.randint(2, 8, (tokens, 1), device="cuda", generator=g)
    where = torch.rand(tokens, experts, device="cuda", generator=g).argsort(-1) < few
    steps = torch.randint(0, 8, (tokens, experts), device="cuda", generator=g)
    logits = torch.where(where, 1 + steps * 2.0 ** -23, logits)
    bias = torch.zeros(experts, device="cuda") if biased else None
    for k in (1, 2, 3, 4):
        _check_route(logits, k, bias=bias, scoring="sigmoid", grad=False)
        _check_route(logits, k, bias=bias, scoring="softmax", grad=False)


def test_route_of_all_experts_that_are_all_out():
    """As many choices as experts, none of them live: nothing behind the last expert is touched."""
    for experts, k in ((31, 31), (9, 9), (5, 5), (33, 31)):
        logits = torch.full((40, experts), -math.inf, device="cuda")
        logits[::2, 0] = 1.0
        for bias in (None, torch.zeros(experts, device="cuda")):
            got = route_topk(logits, k, bias=bias, scoring="sigmoid")
            assert torch.equal(got.idx.long(), torch.arange(k, device="cuda").expand(40, k))
            assert bool((got.weights[1::2] == 0).all()) and bool((got.weights[::2, 0] == 1).all())


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("biased", [False, True])
def test_route_with_infinities_and_nan(scoring, renormalise, biased):
    g = _gen(6)
    logits = _normal(g, 64, 12)
    logits[0] = -math.inf
    logits[1] = math.nan
    logits[2, 3:] = -math.inf                                     # fewer live experts than choices
    logits[3, ::2] = math.nan
    logits[4, 5] = math.inf
    logits[5, 2:4] = math.inf
    logits[6] = torch.finfo(torch.float32).min
    logits[7] = -200.0                                            # scores that underflow
    logits[8] = 200.0
    logits[9, :6] = -math.inf                                     # whole groups out
    bias = 0.1 * _normal(g, 12) if biased else None
    finite = dict(scoring=scoring, renormalise=renormalise)
    got = route_topk(logits, 4, bias=bias, **finite)
    idx, rows, offsets = ref.route(logits, 4, bias, scoring)
    if biased and scoring == "softmax":                           # row 6: 64 bits and 32 agree that all are equal
        assert torch.equal(got.idx[:, 0].long(), idx[:, 0])
    assert torch.equal(got.idx.long(), idx) and torch.equal(got.rows.long(), rows) and torch.equal(got.offsets.long(), offsets)
    assert bool(torch.isfinite(got.weights).all())
    want = ref.weights(ref.clean(logits), idx, scoring, renormalise, 1.0)
    dead = ref.clean(logits).amax(-1) == -math.inf
    torch.testing.assert_close(got.weights[~dead].double(), want[~dead], rtol=2 ** -14, atol=2 ** -126)
    assert bool((got.weights[dead] == 0).all())
    leaf = logits.clone().requires_grad_(True)
    dl, = torch.autograd.grad(route_topk(leaf, 4, bias=bias, **finite).weights, leaf, torch.ones(64, 4, device="cuda"))
    assert bool(torch.isfinite(dl).all()) and bool((dl[~torch.isfinite(logits) & (logits != math.inf)] == 0).all())
    for group_score in ("max", "top2"):
        got = route_topk(logits, 4, bias=bias, groups=4, top_groups=2, group_score=group_score, **finite)
        idx, _, _ = ref.route(logits, 4, bias, scoring, 4, 2, group_score)
        assert torch.equal(got.idx.long(), idx)


def test_route_bias_of_infinities():
    g = _gen(8)
    logits = _normal(g, 100, 16)
    bias = 0.1 * _normal(g, 16)
    bias[3], bias[4], bias[5] = -math.inf, math.inf, math.nan
    got = route_topk(logits, 4, bias=bias, scoring="sigmoid")
    idx, _, _ = ref.route(logits, 4, bias, "sigmoid")
    assert torch.equal(got.idx.long(), idx) and bool((got.idx[:, 0] == 4).all())
    assert not bool(((got.idx == 3) | (got.idx == 5)).any())


def test_route_of_no_tokens_and_of_masked_ones():
    got = route_topk(torch.zeros(0, 8, device="cuda", requires_grad=True), 2)
    assert got.idx.shape == (0, 2) and got.offsets.tolist() == [0] * 9
    got.weights.sum().backward()
    got = route_topk(torch.zeros(50, 8, device="cuda"), 2, mask=torch.zeros(50, dtype=torch.bool, device="cuda"))
    assert bool((got.idx == -1).all()) and bool((got.rows == -1).all()) and bool((got.weights == 0).all())
    assert got.offsets.tolist() == [0] * 9


@pytest.mark.parametrize("dtype", TYPES)
def test_route_of_strided_logits(dtype):
    g = _gen(9)
    wide = _normal(g, 300, 50).to(dtype)
    _check_route(wide[:, 3:43], 4)
    _check_route(wide[::2, 1:40], 4, renormalise=False)
    _check_route(_normal(g, 40, 300).to(dtype).t(), 4)
    _check_route(_normal(g, 1, 40).to(dtype).expand(77, 40), 4, grad=False)


def test_route_gradient_against_differences():
    """Directional derivatives of the weights, choice held, by central differences in 64 bits."""
    g = _gen(10)
    for scoring in ("softmax", "sigmoid"):
        for renormalise in (True, False):
            logits = _normal(g, 20, 24).requires_grad_(True)
            got = route_topk(logits, 5, scoring=scoring, renormalise=renormalise, scale=1.7)
            dw, along = _normal(g, 20, 5), _normal(g, 20, 24).double()
            dl, = torch.autograd.grad(got.weights, logits, dw)
            def f(step):
                return (ref.weights(logits.detach().double() + step * along, got.idx.long(), scoring, renormalise, 1.7)
                        * dw.double()).sum(-1)
            slope = (f(1e-4) - f(-1e-4)) / 2e-4
            # differences: 1e-8 of third derivatives of order one; the gradient: 2^-15 of its terms.
            torch.testing.assert_close((dl.double() * along).sum(-1), slope, rtol=1e-4, atol=1e-4)


# --------------------------------------------------------------------------------------- dispatch / combine
def _routing(g, tokens, experts, top_k, live=1.0, requires_grad=False):
    logits = _normal(g, tokens, experts)
    mask = torch.rand(tokens, device="cuda", generator=g) < live if live < 1 else None
    r = route_topk(logits, top_k, mask=mask)
    return Routing(r.idx, r.weights.detach().requires_grad_(requires_grad), r.rows, r.offsets)


def _check_moves(x, y, routing):
    """dispatch(x) and combine(y) with their gradients; x [tokens, hidden], y [tokens * top_k, hidden]."""
    rows, (t, k) = routing.rows.long(), routing.rows.shape
    n, hidden = t * k, x.shape[1]
    live = (rows >= 0) & (rows < n)
    g = _gen(1)

    x = x.detach().requires_grad_(True)
    out = dispatch(x, routing)
    want = torch.zeros(n, hidden, dtype=x.dtype, device="cuda")
    want[rows[live]] = x.detach()[:, None].expand(t, k, hidden)[live]
    used = torch.zeros(n, dtype=torch.bool, device="cuda")
    used[rows[live]] = True
    assert torch.equal(out.detach()[used], want[used])
    assert bool((out.detach()[int(routing.offsets[-1]):] == 0).all())
    dout = _normal(g, n, hidden).to(x.dtype)
    dx, = torch.autograd.grad(out, x, dout)
    parts = torch.where(live[..., None], dout.double()[rows.clamp(0, n - 1)], 0.0)
    _close(dx, parts.sum(1), k * 2 ** -24 * parts.abs().sum(1), "dispatch dx")

    y = y.detach().requires_grad_(True)
    out = combine(y, routing)
    w = torch.where(live, routing.weights.detach().double(), 0.0)
    parts = w[..., None] * y.detach().double()[rows.clamp(0, n - 1)]
    parts = torch.where(live[..., None], parts, 0.0)
    _close(out.detach(), parts.sum(1), (k + 1) * 2 ** -24 * parts.abs().sum(1), "combine")
    dout = _normal(g, t, hidden).to(y.dtype)
    dy, dw = torch.autograd.grad(out, (y, routing.weights), dout)
    want = torch.zeros(n, hidden, dtype=torch.float64, device="cuda")
    want[rows[live]] = (w[..., None] * dout.double()[:, None])[live]
    _close(dy[used], want[used], 2 ** -24 * want[used].abs(), "combine dy")
    assert bool((dy[int(routing.offsets[-1]):] == 0).all())
    parts = y.detach().double()[rows.clamp(0, n - 1)] * dout.double()[:, None]
    parts = torch.where(live[..., None], parts, 0.0)
    _close(dw, parts.sum(-1), (hidden / 32 + 16) * 2 ** -24 * parts.abs().sum(-1), "combine dweights")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,hidden,experts,top_k,live", [
    (1, 1, 1, 1, 1.0), (1, 4096, 8, 2, 1.0), (7, 33, 8, 3, 1.0), (300, 512, 16, 8, 1.0), (333, 1431, 60, 5, 0.8),
    (50, 7, 8, 8, 0.5), (1025, 2056, 8, 2, 0.9), (64, 8200, 128, 31, 1.0), (3, 20001, 4, 1, 1.0), (200, 100, 9, 9, 0.0), (5000, 8, 8, 2, 0.9), (3001, 64, 16, 6, 1.0), (2500, 200, 8, 3, 0.9),
    (700, 1, 4, 4, 1.0)])
def test_dispatch_and_combine(tokens, hidden, experts, top_k, live, dtype):
    g = _gen(tokens + hidden)
    routing = _routing(g, tokens, experts, top_k, live, requires_grad=True)
    _check_moves(_normal(g, tokens, hidden).to(dtype), _normal(g, tokens * top_k, hidden).to(dtype), routing)


@pytest.mark.parametrize("dtype", TYPES)
def test_moves_of_strided_rows(dtype):
    g = _gen(2)
    routing = _routing(g, 40, 8, 3, requires_grad=True)
    x, y = _normal(g, 40, 300).to(dtype), _normal(g, 120, 300).to(dtype)
    for cut in (slice(0, 256), slice(8, 264), slice(1, 257), slice(5, 130)):
        _check_moves(x[:, cut], y[:, cut], routing)
    _check_moves(_normal(g, 64, 40).to(dtype).t(), _normal(g, 64, 120).to(dtype).t(), routing)
    _check_moves(_normal(g, 1, 64).to(dtype).expand(40, 64), _normal(g, 240, 64).to(dtype)[::2], routing)


def test_moves_of_no_tokens():
    routing = Routing(*(torch.zeros(0, 2, dtype=d, device="cuda") for d in (torch.int32, torch.float32, torch.int32)),
                      torch.zeros(9, dtype=torch.int32, device="cuda"))
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    assert dispatch(x, routing).shape == (0, 16) and combine(x, routing).shape == (0, 16)
    (dispatch(x, routing).sum() + combine(x, routing).sum()).backward()
    assert x.grad.shape == (0, 16)


def test_rows_outside_the_batch_move_nothing():
    """Row numbers from elsewhere: those outside are skipped in every direction (checked by the kernels themselves)."""
    g = _gen(3)
    routing = _routing(g, 30, 8, 2, requires_grad=True)
    rows = routing.rows.clone()
    rows[0, 0], rows[1, 1], rows[2, 0], rows[3, 0] = -7, 60, 2 ** 31 - 1, -2 ** 31
    for hidden in (64, 33):
        _check_moves(_normal(g, 30, hidden), _normal(g, 60, hidden), routing._replace(rows=rows))
    wild = torch.full((9,), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    dispatch(_normal(g, 30, 64), routing._replace(offsets=wild))              # no tail
    out = dispatch(_normal(g, 30, 64), routing._replace(offsets=-wild))       # all of it is tail or written
    torch.cuda.synchronize()
    assert out.shape == (60, 64)


def test_moved_nan_and_infinity_stay_in_their_rows():
    g = _gen(4)
    routing = _routing(g, 20, 8, 2, 0.5)
    x = _normal(g, 20, 64)
    x[3] = math.nan
    x[4] = math.inf
    x[routing.rows[:, 0] < 0] = math.nan                                      # padding tokens
    out = dispatch(x, routing)
    n = int(routing.offsets[-1])
    assert bool((out[n:] == 0).all())
    y = _normal(g, 40, 64)
    y[n:] = math.nan                                                          # rows that no choice reads
    assert bool(torch.isfinite(combine(y, routing)).all())


# ----------------------------------------------------------------------------------------------------- norms
def _check_norm(residual, x, gamma, post, gate, scale=1.0, eps=1e-5, use=("y", "h")):
    leaves = {n: t.detach().requires_grad_(True) for n, t in
              dict(residual=residual, x=x, gamma=gamma, post=post, gate=gate).items() if t is not None}
    L = leaves.get
    if x is None:
        y, h = rms_norm(L("residual"), L("gamma"), eps), None
    else:
        y, h = residual_rms_norm(L("residual"), L("x"), L("gamma"), post_gamma=L("post"), gate=L("gate"),
                                 residual_scale=scale, eps=eps)
    v = {n: t.detach().double().requires_grad_(True) for n, t in leaves.items()}
    V = v.get
    hidden = residual.shape[-1]
    n = residual.numel() // hidden
    flat = lambda t: t.reshape(n, hidden)
    if x is None:
        wy, wh = ref.rms(V("residual"), V("gamma"), eps), V("residual")
    else:
        wy, wh = ref.block_norm(flat(V("residual")), flat(V("x")), V("gamma"), V("post"), V("gate"), scale, eps)
        wy, wh = wy if wy is None else wy.view(residual.shape), wh.view(residual.shape)
    with torch.no_grad():
        # A root: (16 + 10) / 2 roundings of a sum of squares, rsqrtf and two products, below 2^-19; a value of v,
        # h or y after at most four such factors: 2^-17 of what it is made of.
        u = V("x") if x is not None else torch.zeros_like(wh)
        r1 = torch.rsqrt(flat(u).square().mean(-1, keepdim=True) + eps)
        n1 = flat(u) * r1
        after = flat(u) if post is None else n1 * V("post")
        gates = torch.ones(1, hidden, device="cuda", dtype=torch.float64) if gate is None else \
            V("gate").view(-1, 1, hidden).expand(-1, max(1, n // V("gate").view(-1, hidden).shape[0]), hidden).reshape(-1, hidden)[:max(n, 1)]
        made = flat(V("residual")).abs() * abs(scale) + (after * gates).abs()
        r2 = torch.rsqrt(flat(wh).square().mean(-1, keepdim=True) + eps)
        rough = made.square().mean(-1, keepdim=True).sqrt() * r2         # above 1 where h cancels
        if h is not None:
            assert h.dtype == residual.dtype and h.shape == residual.shape
            _close(flat(h.detach()), flat(wh.detach()), 2 ** -17 * made, "h")
        if gamma is not None:
            assert y.dtype == (x if x is not None else residual).dtype and y.shape == residual.shape
            _close(flat(y.detach()), flat(wy.detach()), 2 ** -16 * V("gamma").abs() * r2 * (made + flat(wh).abs() * rough), "y")
    ends = [(t, w) for name, t, w in (("y", y, wy), ("h", h, wh)) if t is not None and name in use]
    g = _gen(7)
    back = [_normal(g, *residual.shape).to(t.dtype) for t, _ in ends]
    grads = dict(zip(leaves, torch.autograd.grad([t for t, _ in ends], list(leaves.values()), back, allow_unused=True)))
    wants = dict(zip(leaves, torch.autograd.grad([w for _, w in ends], list(v.values()), [b.double() for b in back], allow_unused=True)))
    with torch.no_grad():
        # Sizes of the terms that each gradient is made of; each is off by 2^-15 of them.
        dy = next((flat(b.double()) for (t, _), b in zip(ends, back) if t is y), torch.zeros(n, hidden, device="cuda", dtype=torch.float64))
        dh = next((flat(b.double()) for (t, _), b in zip(ends, back) if t is h), torch.zeros_like(dy))
        n2 = made * r2
        a = (dy * V("gamma")).abs() if gamma is not None else torch.zeros_like(dy)
        d = dh.abs() + r2 * (a + n2 * rough * (a * n2).mean(-1, keepdim=True))
        dv = d * gates.abs()
        b = dv * V("post").abs() if post is not None else dv
        dx = r1 * (b + n1.abs() * (b * n1.abs()).mean(-1, keepdim=True)) if post is not None else dv
        size = dict(residual=abs(scale) * d, x=dx, gamma=(dy.abs() * n2 * rough).sum(0), post=(dv * n1.abs()).sum(0))
        if gate is not None:
            size["gate"] = (d * after.abs()).view(-1, max(1, n // V("gate").view(-1, hidden).shape[0]), hidden).sum(1).view(gate.shape) \
                if n else torch.zeros(gate.shape, device="cuda", dtype=torch.float64)
        for name, want in wants.items():
            if want is None:
                assert grads[name] is None or bool((grads[name] == 0).all())
                continue
            assert grads[name].dtype == leaves[name].dtype
            rows = name in ("residual", "x")
            # Sums over n rows add n 2^-24, in strips of n / 296 + 37 + 8 terms: below 2^-15 up to 2^17 rows.
            _close(flat(grads[name]) if rows else grads[name], flat(want) if rows else want,
                   (2 ** -15 if rows else 2 ** -14) * size[name], f"d{name}")


NORMS = [
    # rows shape, hidden, pre, post, gates (0 none, 1 one, more: sequences), scale
    ((1,), 1, True, True, 1, 1.0), ((1,), 4096, True, False, 0, 1.0), ((8,), 4096, True, True, 8, 0.9),
    ((3, 5), 64, True, True, 3, 1.0), ((40,), 33, True, True, 5, 0.5), ((1000,), 96, True, False, 0, 1.0),
    ((999,), 513, True, True, 1, 1.0), ((700,), 1000, False, True, 7, 2.0), ((602,), 2055, True, True, 2, 1.0),
    ((301,), 4096, False, False, 1, 1.0), ((6, 100), 2048, True, True, 6, 0.9), ((64,), 8192, True, True, 64, 1.0),
    ((37,), 16384, True, True, 1, 1.0), ((9,), 16383, True, True, 3, 1.0), ((2000,), 256, False, False, 0, 0.7),
    ((5000,), 136, True, True, 4, 1.0), ((400,), 8200, True, True, 4, 1.0), ((333,), 12289, True, True, 9, 0.9),
    ((500,), 10240, True, False, 0, 1.0), ((211,), 16384, True, True, 211, 1.0), ((300,), 9001, False, True, 0, 1.0),
]


@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.float16, torch.float16),
                                   (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                   (torch.float16, torch.float32)], ids=str)
@pytest.mark.parametrize("case", NORMS, ids=lambda c: "x".join(map(str, c[0])) + f"x{c[1]}g{c[4]}")
def test_residual_rms_norm(case, types):
    shape, hidden, pre, post, gates, scale = case
    xt, rt = types
    g = _gen(hidden + shape[0])
    x, residual = (1.5 * _normal(g, *shape, hidden)).to(xt), (2 * _normal(g, *shape, hidden)).to(rt)
    gamma = (1 + 0.1 * _normal(g, hidden)).to(xt) if pre else None
    post_gamma = (1 + 0.1 * _normal(g, hidden)).to(xt) if post else None
    gate = (0.5 + 0.2 * _normal(g, *((gates, hidden) if gates > 1 else (hidden,)))).to(xt) if gates else None
    _check_norm(residual, x, gamma, post_gamma, gate, scale)


@pytest.mark.parametrize("use", [("y",), ("h",)])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("rt", [torch.bfloat16, torch.float32])
def test_norm_gradients_of_one_output_and_32_bit_weights(use, post, rt):
    g = _gen(12)
    for hidden in (512, 77):
        x, residual = _normal(g, 130, hidden).bfloat16(), _normal(g, 130, hidden).to(rt)
        w = [1 + 0.1 * _normal(g, hidden) for _ in range(3)]
        _check_norm(residual, x, w[0], w[1] if post else None, w[2] if post else None, 1.0, use=use)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,hidden", [(1, 1), (5, 4096), (1000, 320), (33, 16384), (77, 1023)])
def test_rms_norm(rows, hidden, dtype):
    g = _gen(rows)
    _check_norm(_normal(g, rows, hidden).to(dtype), None, (1 + 0.1 * _normal(g, hidden)).to(dtype), None, None)


def test_norm_of_one_tensor_twice():
    g = _gen(18)
    x = _normal(g, 70, 320).bfloat16().requires_grad_(True)
    gamma = (1 + 0.1 * _normal(g, 320)).bfloat16()
    y, h = residual_rms_norm(x, x, gamma)
    dy, dh = _normal(g, 70, 320).bfloat16(), _normal(g, 70, 320).bfloat16()
    both, = torch.autograd.grad((y, h), x, (dy, dh))
    a, b = x.detach().clone().requires_grad_(True), x.detach().clone().requires_grad_(True)
    parts = torch.autograd.grad(residual_rms_norm(a, b, gamma), (a, b), (dy, dh))
    assert torch.equal(both, parts[0] + parts[1])
    y, h = residual_rms_norm(x, x, gamma)
    (y.float().sum() + h.float().sum()).backward()
    assert x.grad.shape == x.shape


def test_norm_of_zero_rows_and_rows_of_zeros():
    g = _gen(13)
    gamma, gate = torch.ones(64, device="cuda", requires_grad=True), torch.ones(2, 64, device="cuda", requires_grad=True)
    x = torch.zeros(0, 64, device="cuda", requires_grad=True)
    y, h = residual_rms_norm(x, x, gamma, post_gamma=gamma, gate=gate)
    (y.sum() + h.sum()).backward()
    assert x.grad.shape == (0, 64) and bool((gamma.grad == 0).all()) and bool((gate.grad == 0).all())
    zeros = torch.zeros(6, 64, device="cuda")
    _check_norm(zeros, zeros, 1 + 0.1 * _normal(g, 64), 1 + 0.1 * _normal(g, 64), None)
    y, _ = residual_rms_norm(zeros, zeros, torch.ones(64, device="cuda"), eps=0.0)
    assert bool(y.isnan().all())                                   # 0 / 0, as the formula has it


def test_norm_nan_stays_in_its_row():
    g = _gen(14)
    x, residual = _normal(g, 50, 128), _normal(g, 50, 128)
    gamma = 1 + 0.1 * _normal(g, 128)
    y0, h0 = residual_rms_norm(residual, x, gamma, post_gamma=gamma)
    x[7, 3], residual[9, 100] = math.nan, math.inf
    y1, h1 = residual_rms_norm(residual, x, gamma, post_gamma=gamma)
    keep = torch.ones(50, dtype=torch.bool, device="cuda")
    keep[7] = keep[9] = False
    assert torch.equal(y0[keep], y1[keep]) and torch.equal(h0[keep], h1[keep]) and bool(y1[7].isnan().all())


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_strided_rows(dtype):
    g = _gen(15)
    wide = [_normal(g, 40, 700).to(dtype) for _ in range(2)]
    gamma = (1 + 0.1 * _normal(g, 700)).to(dtype)
    for cut in (slice(0, 512), slice(8, 520), slice(1, 513), slice(3, 334)):
        w = gamma[cut]
        _check_norm(wide[0][:, cut], wide[1][:, cut], w, w, w)
    _check_norm(wide[0][:, :40].t(), wide[1][::1, :40].t(), gamma[:40], None, None)
    _check_norm(wide[0][:, :660].view(40, 1, 660).expand(40, 2, 660)[:, :, ::2], wide[1][:, :660].view(40, 2, 330), gamma[:660:2], None, None)


def test_norm_gradient_against_differences():
    g = _gen(16)
    names = ("residual", "x", "gamma", "post", "gate")
    leaves = [_normal(g, 12, 40), _normal(g, 12, 40), 1 + 0.1 * _normal(g, 40), 1 + 0.1 * _normal(g, 40), _normal(g, 3, 40)]
    leaves = [t.requires_grad_(True) for t in leaves]
    y, h = residual_rms_norm(leaves[0], leaves[1], leaves[2], post_gamma=leaves[3], gate=leaves[4], residual_scale=0.8)
    dy, dh = _normal(g, 12, 40), _normal(g, 12, 40)
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))
    for i, name in enumerate(names):
        along = _normal(g, *leaves[i].shape).double()

        def f(step):
            v = [t.detach().double() + (step * along if j == i else 0) for j, t in enumerate(leaves)]
            wy, wh = ref.block_norm(*v, 0.8, 1e-5)
            return (wy * dy.double()).sum() + (wh * dh.double()).sum()

        # 1e-10 of third derivatives; the gradient's own 2^-15 of terms whose sizes add up to about a thousand.
        slope = (f(1e-5) - f(-1e-5)) / 2e-5
        assert abs(float((grads[i].double() * along).sum() - slope)) <= 2 ** -15 * float((grads[i].double() * along).abs().sum()) * 8 + 1e-4, name


# ------------------------------------------------------------------------------------- as a user's program has them
def _step(logits, x, stream, gamma, gate):
    """One pass of everything and its gradients."""
    r = route_topk(logits, 3, scoring="sigmoid", groups=2, top_groups=1, bias=torch.zeros(16, device="cuda"))
    out = combine(dispatch(x, r) * 2, r)
    y, h = residual_rms_norm(stream, out, gamma, post_gamma=gamma, gate=gate, residual_scale=0.5)
    grads = torch.autograd.grad((y.float().square().sum() + h.float().sum()), (logits, x, stream, gamma, gate))
    return (r.idx, r.weights.detach(), r.rows, r.offsets, y.detach(), h.detach()) + grads


def _inputs(seed, tokens=300, hidden=256):
    g = _gen(seed)
    return [t.requires_grad_(True) for t in (
        _normal(g, tokens, 16), _normal(g, tokens, hidden).bfloat16(), _normal(g, tokens, hidden).bfloat16(),
        (1 + 0.1 * _normal(g, hidden)).bfloat16(), _normal(g, 2, hidden).bfloat16())]


def test_results_do_not_change_from_run_to_run():
    args = _inputs(1, tokens=9000)
    first = _step(*args)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _step(*args)))


def test_two_streams_at_once():
    args = [_inputs(s, tokens=5000) for s in (1, 2)]
    want = [_step(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [None, None]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _step(*args[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(want[i], got[i]))


def test_long_rows_captured():
    """Rows that two blocks share, forward and backward, captured and replayed on other inputs."""
    def make(seed):
        g = _gen(seed)
        return [t.requires_grad_(True) for t in (_normal(g, 300, 9216).bfloat16(), _normal(g, 300, 9216).bfloat16(),
                                                 (1 + 0.1 * _normal(g, 9216)).bfloat16(), _normal(g, 3, 9216).bfloat16())]

    def step(stream, x, gamma, gate):
        y, h = residual_rms_norm(stream, x, gamma, post_gamma=gamma, gate=gate)
        return torch.autograd.grad(y.float().square().sum() + h.float().sum(), (stream, x, gamma, gate))

    args = make(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*args)
    fresh = make(2)
    for a, b in zip(args, fresh):
        a.data.copy_(b.data)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, step(*fresh)))


def test_two_captured_graphs():
    """Forward and backward captured twice, replayed in turn and on other inputs."""
    sets = [_inputs(s) for s in (1, 2)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for args in sets:
            _step(*args)
    torch.cuda.current_stream().wait_stream(side)
    for args in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(*args))
        graphs.append(graph)
    for seed in (5, 6):
        fresh = [_inputs(seed + 10 * i) for i in range(2)]
        for args, new in zip(sets, fresh):
            for a, b in zip(args, new):
                a.data.copy_(b.data)
        for graph in graphs + graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, new in zip(outs, fresh):
            assert all(torch.equal(a, b) for a, b in zip(out, _step(*new)))


def test_gradients_are_taken_once():
    args = _inputs(3)
    r = route_topk(args[0], 2)
    for leaf, out in ((args[0], r.weights), (args[1], dispatch(args[1], r)), (args[3], rms_norm(args[2], args[3])),
                      (args[0], combine(torch.ones(600, 8, device="cuda"), r))):
        grad, = torch.autograd.grad(out.float().square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            grad.float().square().sum().backward()


def test_changed_inputs_are_noticed():
    args = _inputs(4)
    y, h = residual_rms_norm(args[2], args[1] * 1, args[3])
    with torch.no_grad():
        args[2].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        (y.sum() + h.sum()).backward()


def test_more_than_2_to_the_31_values():
    """Offsets beyond 31 bits: a wide batch of tokens through every operator, checked at both ends and between."""
    tokens, hidden = 160_001, 16384                                # 2.6e9 values, 5.2 GB
    x = torch.empty(tokens, hidden, dtype=torch.bfloat16, device="cuda")
    for i in range(0, tokens, 20000):
        x[i:i + 20000] = torch.randn(min(20000, tokens - i), hidden, device="cuda", generator=_gen(i)).bfloat16()
    at = torch.tensor([0, 1, 65535, 131071, 131073, tokens - 2, tokens - 1], device="cuda")
    gamma = torch.ones(hidden, dtype=torch.bfloat16, device="cuda")
    y, h = residual_rms_norm(x, x, gamma)
    wy, wh = residual_rms_norm(x[at], x[at], gamma)
    assert torch.equal(y[at], wy) and torch.equal(h[at], wh)
    del y, h
    r = route_topk(torch.randn(tokens, 8, device="cuda", generator=_gen(1)), 1)
    out = dispatch(x, r)
    assert torch.equal(out[r.rows[at, 0].long()], x[at])
    back = combine(out, r)
    assert torch.equal(back[at], x[at])
    del out, back, x
    logits = torch.empty(2_200_003, 1024, dtype=torch.bfloat16, device="cuda")
    for i in range(0, logits.shape[0], 200_000):
        logits[i:i + 200_000] = torch.randn(min(200_000, logits.shape[0] - i), 1024, device="cuda", generator=_gen(i)).bfloat16()
    r = route_topk(logits, 2)
    at = torch.tensor([0, 2 ** 21 - 1, 2 ** 21, 2 ** 21 + 1, logits.shape[0] - 1], device="cuda")
    idx, _, _ = ref.route(logits[at], 2)
    assert torch.equal(r.idx[at].long(), idx) and int(r.offsets[-1]) == 2 * logits.shape[0]
    assert torch.equal(torch.bincount(r.idx.flatten().long(), minlength=1024), (r.offsets[1:] - r.offsets[:-1]).long())


@pytest.mark.parametrize("how", [dict(), dict(scoring="sigmoid", groups=4, top_groups=2, group_score="top2", scale=2.5)])
@pytest.mark.parametrize("masked", [False, True])
def test_sparse_moe_blocks_in_a_row(how, masked):
    """Two blocks as a model has them, in 32 bits, against the same formulas in 64: outputs and every gradient."""
    from pccl_b200.models import SparseMoEBlock
    torch.manual_seed(0)
    tokens, hidden, ffn, experts, top_k = 200, 64, 96, 16, 4
    blocks = [SparseMoEBlock(hidden, ffn, experts, top_k, post_norm=True, gated=True, balance=bool(how), residual_scale=0.9,
                             dtype=torch.float32, **how) for _ in range(2)]
    final = torch.nn.Parameter(torch.ones(hidden, device="cuda"))
    x = torch.randn(tokens, hidden, device="cuda", requires_grad=True)
    mask = torch.rand(tokens, device="cuda") < 0.8 if masked else None
    normed, stream = blocks[0](x, next_gamma=blocks[1].gamma, mask=mask)
    normed, stream = blocks[1](stream, normed=normed, next_gamma=final, mask=mask)
    back = torch.randn(tokens, hidden, device="cuda")
    ((normed * back).sum() + stream.sum()).backward()

    leaves = {}

    def wide(name, p):
        leaves[name] = p.detach().double().requires_grad_(True)
        return leaves[name]

    s = wide("x", x)
    for i, b in enumerate(blocks):
        p = {n: wide(f"{i}.{n}", t) for n, t in b.named_parameters()}
        n = ref.rms(s, p["gamma"], b.eps)
        logits = n @ p["wg"].t()
        idx, _, _ = ref.route(logits.detach(), top_k, b.bias, how.get("scoring", "softmax"), how.get("groups", 1),
                              how.get("top_groups"), how.get("group_score", "max"), mask)
        w = ref.weights(logits, idx, how.get("scoring", "softmax"), True, how.get("scale", 1.0))
        out = torch.zeros_like(n)
        for e in range(experts):
            gate, up = (n @ p["w13"][e].t()).chunk(2, dim=-1)
            out = out + (torch.nn.functional.silu(gate) * up @ p["w2"][e].t()) * torch.where(idx == e, w, 0.0).sum(-1, keepdim=True)
        _, s = ref.block_norm(s, out, None, p["post_gamma"], p["gate"], 0.9, b.eps)
    f = wide("final", final)
    y = ref.rms(s, f, 1e-5)
    ((y * back.double()).sum() + s.sum()).backward()
    # 32-bit chains of about a thousand roundings through two blocks, library products (tf32 off) among them.
    torch.testing.assert_close(normed.double(), y.detach(), rtol=1e-3, atol=1e-3)
    torch.testing.assert_close(stream.double(), s.detach(), rtol=1e-3, atol=1e-3)
    own = {"x": x, "final": final, **{f"{i}.{n}": t for i, b in enumerate(blocks) for n, t in b.named_parameters()}}
    for name, t in own.items():
        want = leaves[name].grad
        assert float((t.grad.double() - want).norm()) <= 1e-3 * float(want.norm()) + 1e-6, name
