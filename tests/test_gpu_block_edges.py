"""Routing, dispatch / combine and the block norms on the GPU where they can go wrong: sums that cancel, choices
that are left out.  Tolerances as in test_gpu_block_ops.py; what is not rounded is compared bit by bit."""

import copy
import io
import math

import pytest
import torch

import block_reference as ref
from block_reference import HALF_STEP, TINY
from pccl_b200.ops import Routing, combine, dispatch, route_topk

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


# ------------------------------------------------------------------------------------------------- routing
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("size", [16.0, 512.0, 4096.0])
@pytest.mark.parametrize("experts,groups,top_groups,top_k", [
    (8, 4, 2, 3), (16, 8, 4, 5), (64, 8, 3, 4), (256, 8, 4, 8), (42, 6, 3, 3), (512, 32, 16, 8), (1000, 20, 7, 9)])
def test_route_groups_whose_best_two_cancel(experts, groups, top_groups, top_k, size, scoring):
    """A group's two best biased scores are near +size and -size: their sum has lost what 32 bits of either lose."""
    g = _gen(experts)
    each, tokens = experts // groups, 30000 if experts <= 64 else 6000
    bias = torch.full((groups, each), -2 * size, device="cuda")
    bias[:, 0], bias[:, 1] = size, -size
    bias = bias.flatten()
    logits = 0.7 * _normal(g, tokens, experts)
    got = route_topk(logits, top_k, bias=bias, scoring=scoring, groups=groups, top_groups=top_groups, group_score="top2")
    idx, rows, offsets = ref.route(logits, top_k, bias, scoring, groups, top_groups, "top2")
    wrong = (got.idx.long() != idx).any(-1)
    assert not bool(wrong.any()), f"{int(wrong.sum())} of {tokens} tokens"
    assert torch.equal(got.rows.long(), rows) and torch.equal(got.offsets.long(), offsets)


# --------------------------------------------------------------------------------------- dispatch / combine
def _leave_nan_behind(*sizes):
    """Fills the memory that the next allocations of these sizes (in bytes) are made of with NaN."""
    held = [torch.full((max(1, n // 4),), math.nan, device="cuda") for n in sizes for _ in range(3)]
    torch.cuda.synchronize()
    del held


def _dropped(g, tokens, experts, top_k, capacity, live):
    """A routing whose choices beyond `capacity` rows an expert are left out, as a layer with bounded experts does."""
    mask = torch.rand(tokens, device="cuda", generator=g) < live if live < 1 else None
    r = route_topk(_normal(g, tokens, experts), top_k, mask=mask)
    place = r.rows - r.offsets[:-1][r.idx.clamp(min=0).long()]
    rows = torch.where((r.idx >= 0) & (place < capacity), r.rows, -1).contiguous()
    return Routing(r.idx, r.weights.detach().requires_grad_(True), rows, r.offsets)


def _check_whole(x, y, routing):
    """dispatch(x), the gradient of combine(y): every row, those that no choice names among them."""
    rows, (t, k) = routing.rows.long(), routing.rows.shape
    n, hidden = t * k, x.shape[1]
    live = (rows >= 0) & (rows < n)
    named = torch.zeros(n, dtype=torch.bool, device="cuda")
    named[rows[live]] = True
    want = torch.zeros(n, hidden, dtype=x.dtype, device="cuda")
    want[rows[live]] = x[:, None].expand(t, k, hidden)[live]
    nbytes = n * hidden * x.element_size()
    _leave_nan_behind(nbytes)
    out = dispatch(x, routing)
    assert torch.equal(out, want), f"{int((out != want).any(-1).sum())} rows of {n}, {int(named.sum())} named"
    y = y.detach().requires_grad_(True)
    dout = _normal(_gen(1), t, hidden).to(y.dtype)
    out = combine(y, routing)
    _leave_nan_behind(nbytes)
    dy, dw = torch.autograd.grad(out, (y, routing.weights), dout)
    w = torch.where(live, routing.weights.detach().double(), 0.0)
    wide = torch.zeros(n, hidden, dtype=torch.float64, device="cuda")
    wide[rows[live]] = (w[..., None] * dout.double()[:, None])[live]
    # one product in 32 bits, rounded once more to the type
    off = (dy.double() - wide).abs()
    assert bool((off <= HALF_STEP[y.dtype] * wide.abs() * (1 + 2 ** -10) + TINY[y.dtype] + 2 ** -24 * wide.abs()).all())
    assert bool((dy[~named] == 0).all()) and bool((dw[~live] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,hidden,experts,top_k,capacity,live", [
    (1, 64, 4, 1, 0, 1.0), (8, 4096, 8, 2, 1, 1.0), (64, 33, 8, 2, 9, 0.8), (500, 256, 16, 2, 40, 1.0),
    (300, 1431, 8, 3, 70, 0.9), (1000, 1, 4, 1, 100, 1.0), (4000, 128, 8, 2, 700, 1.0), (4096, 511, 16, 4, 900, 0.5),
    (9000, 2056, 8, 8, 8000, 1.0), (3000, 64, 8, 2, 0, 1.0)])
def test_rows_of_left_out_choices_are_zero(tokens, hidden, experts, top_k, capacity, live, dtype):
    g = _gen(tokens + hidden)
    routing = _dropped(g, tokens, experts, top_k, capacity, live)
    _check_whole(_normal(g, tokens, hidden).to(dtype), _normal(g, tokens * top_k, hidden).to(dtype), routing)


def test_rows_named_from_elsewhere_leave_zeros():
    """Row numbers outside the batch, and offsets that say something else than the rows: the rows alone count."""
    g = _gen(3)
    for tokens in (30, 3000):
        r = route_topk(_normal(g, tokens, 8), 2)
        rows = r.rows.clone()
        rows[0, 0], rows[1, 1], rows[2, 0], rows[3, 0] = -7, 2 * tokens, 2 ** 31 - 1, -2 ** 31
        for offsets in (r.offsets, torch.zeros_like(r.offsets), torch.full_like(r.offsets, 2 ** 31 - 1)):
            routing = Routing(r.idx, r.weights.detach().requires_grad_(True), rows, offsets)
            for hidden in (64, 33):
                _check_whole(_normal(g, tokens, hidden), _normal(g, 2 * tokens, hidden), routing)


def test_moves_captured_with_choices_left_out():
    """Enough choices for the kernel that notes them, captured and replayed with other rows and other values."""
    g = _gen(5)
    r = [_dropped(g, 1500, 8, 2, c, 0.9) for c in (1000, 300, 50)]
    rows, weights = r[0].rows.clone(), r[0].weights.detach().clone().requires_grad_(True)
    x = _normal(g, 1500, 136).bfloat16().requires_grad_(True)

    def step(x, weights, rows):
        routing = Routing(r[0].idx, weights, rows, r[0].offsets)
        out = dispatch(x, routing)
        back = combine(out * 2, routing)
        return (out.detach(), back.detach()) + torch.autograd.grad(back.float().square().sum(), (x, weights))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, weights, rows)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(x, weights, rows)
    for new in r[1:] + r[:1]:
        with torch.no_grad():
            x.copy_(_normal(g, 1500, 136))
            rows.copy_(new.rows)
            weights.copy_(new.weights)
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        fresh = step(x.detach().clone().requires_grad_(True), weights.detach().clone().requires_grad_(True), rows.clone())
        assert all(torch.equal(a, b) for a, b in zip(outs, fresh))
        dead = torch.ones(3000, dtype=torch.bool, device="cuda")
        dead[rows[rows >= 0].long()] = False
        assert bool((outs[0][dead] == 0).all())


# ------------------------------------------------------------------------------------- as a user's program has them
@pytest.mark.parametrize("tokens", [1, 5000])
def test_a_routing_is_saved_and_copied(tokens):
    """All of a routing in one file, as a program does that replays one, with no more bytes than it has; and a deep copy."""
    r = route_topk(_normal(_gen(7), tokens, 64), 4)
    file = io.BytesIO()
    torch.save(r, file)
    assert len(file.getvalue()) < tokens * 4 * 12 + 65 * 4 + 16384
    file.seek(0)
    for copied in (torch.load(file, weights_only=False), copy.deepcopy(r)):
        assert type(copied) is Routing
        assert all(torch.equal(a, b) and a.dtype == b.dtype and a.data_ptr() != b.data_ptr() for a, b in zip(copied, r))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens", [0, 40])
def test_block_without_live_tokens_has_every_gradient(tokens, dtype):
    """All tokens masked, and no tokens: every parameter that takes part gets a gradient of the block's type."""
    from pccl_b200.models import SparseMoEBlock
    torch.manual_seed(0)
    block = SparseMoEBlock(64, 96, 8, 2, post_norm=True, gated=True, dtype=dtype)
    x = torch.randn(tokens, 64, device="cuda").to(dtype).requires_grad_(True)
    y, stream = block(x, next_gamma=torch.ones(64, dtype=dtype, device="cuda"),
                      mask=torch.zeros(tokens, dtype=torch.bool, device="cuda"))
    assert torch.equal(stream, x)                                   # nothing is added to the stream
    (y.float().square().sum() + stream.float().sum()).backward()
    for name, p in block.named_parameters():
        assert p.grad is not None and p.grad.dtype == dtype and bool((p.grad == 0).all()), name
    assert x.grad.shape == x.shape


def test_sparse_moe_block_in_its_default_type():
    """bfloat16, as the class is made by default, against the same operators on its own intermediate values: what the block
    wires together.  The library products are the same calls, so the results are equal."""
    from pccl_b200.models import SparseMoEBlock
    from pccl_b200.ops import residual_rms_norm, rms_norm
    torch.manual_seed(1)
    block = SparseMoEBlock(128, 64, 8, 2, post_norm=True, gated=True, balance=True, scoring="sigmoid")
    assert {p.dtype for p in block.parameters()} == {torch.bfloat16}
    x = torch.randn(300, 128, device="cuda").bfloat16().requires_grad_(True)
    gamma = (1 + 0.1 * torch.randn(128, device="cuda")).bfloat16()
    y, stream = block(x, next_gamma=gamma)
    grads = torch.autograd.grad(y.float().square().sum() + stream.float().sum(), [x] + list(block.parameters()))
    n = rms_norm(x, block.gamma)
    r = route_topk(n.float() @ block.wg.float().t(), 2, bias=block.bias, scoring="sigmoid")
    rows, ends = dispatch(n, r), r.offsets.tolist()
    parts = []
    for e in range(8):
        gate, up = (rows[ends[e]:ends[e + 1]] @ block.w13[e].t()).chunk(2, dim=-1)
        parts.append((torch.nn.functional.silu(gate) * up) @ block.w2[e].t())
    wy, ws = residual_rms_norm(x, combine(torch.cat(parts), r), gamma, post_gamma=block.post_gamma, gate=block.gate)
    assert torch.equal(y, wy) and torch.equal(stream, ws)
    wants = torch.autograd.grad(wy.float().square().sum() + ws.float().sum(), [x] + list(block.parameters()))
    for (name, _), got, want in zip([("x", x)] + list(block.named_parameters()), grads, wants):
        assert torch.equal(got, want) and got.dtype == torch.bfloat16 and bool((got != 0).any()), name


def test_calls_in_inference_mode_and_under_vmap():
    """Inference mode gives the same results; a batched tensor of vmap is refused, not read as something else."""
    from pccl_b200.ops import residual_rms_norm
    g = _gen(6)
    logits, x, gamma = _normal(g, 50, 16), _normal(g, 50, 64).bfloat16(), torch.ones(64, device="cuda")

    def step():
        r = route_topk(logits, 2, bias=torch.zeros(16, device="cuda"))
        return tuple(r) + (out := dispatch(x, r), combine(out, r)) + residual_rms_norm(x, x, gamma)

    want = step()
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(want, step()))
    r = route_topk(logits, 2)
    for call in (lambda t: dispatch(t, r), lambda t: residual_rms_norm(t, t, gamma)[0]):
        with pytest.raises((RuntimeError, ValueError)):
            torch.vmap(call)(x.expand(3, 50, 64))
    with pytest.raises((RuntimeError, ValueError)):
        torch.vmap(lambda t: route_topk(t, 2).weights)(logits.expand(3, 50, 16))
