"""Refusals and host paths of routing, dispatch / combine, the block norms and the trainable block that need no GPU."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from pccl_b200.ops import Routing, combine, dispatch, residual_rms_norm, rms_norm, route_topk


def _routing(weights=None):
    return Routing(torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2) if weights is None else weights,
                   torch.arange(8, dtype=torch.int32).view(4, 2), torch.zeros(9, dtype=torch.int32))


CALLS = {
    "logits": lambda d: route_topk(d(4, 8), 2),
    "bias": lambda d: route_topk(torch.zeros(4, 8), 2, bias=d(8)),
    "dispatch: x": lambda d: dispatch(d(4, 16), _routing()),
    "combine: y": lambda d: combine(d(8, 16), _routing()),
    "routing.weights": lambda d: combine(torch.zeros(8, 16), _routing(d(4, 2))),
    "rms_norm: x": lambda d: rms_norm(d(4, 16), torch.zeros(16)),
    "residual": lambda d: residual_rms_norm(d(4, 16), torch.zeros(4, 16), torch.zeros(16)),
    "residual_rms_norm: x": lambda d: residual_rms_norm(torch.zeros(4, 16), d(4, 16), torch.zeros(16)),
    "gamma": lambda d: residual_rms_norm(torch.zeros(4, 16), torch.zeros(4, 16), d(16)),
    "post_gamma": lambda d: residual_rms_norm(torch.zeros(4, 16), torch.zeros(4, 16), None, post_gamma=d(16)),
    "gate": lambda d: residual_rms_norm(torch.zeros(4, 16), torch.zeros(4, 16), None, gate=d(2, 16)),
}


@pytest.mark.parametrize("what", CALLS)
def test_forward_mode_tangents_are_refused(what):
    """Without this a tensor that carries a tangent, but requires no gradient, would lose it without a word."""
    with fwd.dual_level():
        with pytest.raises(ValueError, match=f"{what} has a forward-mode tangent"):
            CALLS[what](lambda *shape: fwd.make_dual(torch.zeros(shape), torch.ones(shape)))
        with pytest.raises(ValueError, match="CUDA device"):        # a level alone changes nothing
            CALLS[what](lambda *shape: torch.zeros(shape))


def test_forward_mode_and_requires_grad():
    with fwd.dual_level():
        x = fwd.make_dual(torch.zeros(4, 16, requires_grad=True), torch.ones(4, 16))
        with pytest.raises(ValueError, match="forward-mode tangent"):
            dispatch(x, _routing())


@pytest.mark.parametrize("rows", [0, 6])
def test_experts_without_rows_still_have_gradients(rows):
    """A batch whose tokens are all masked, or that has none: gradients of zero, not none at all.  With none, ranks that
    average them would not agree on what there is to reduce."""
    from pccl_b200.models import SparseMoEBlock
    block = SparseMoEBlock(16, 32, 4, 2, dtype=torch.float32, device="cpu")
    x = torch.randn(rows, 16, requires_grad=True)
    out = block.experts(x, torch.zeros(5, dtype=torch.int32))
    assert out.shape == (rows, 16) and bool((out == 0).all())
    out.sum().backward()
    for t in (block.w13, block.w2, x):
        assert t.grad is not None and t.grad.shape == t.shape and bool((t.grad == 0).all())


def test_experts_on_their_rows():
    """Some experts without rows, some rows unused, against each row's own products."""
    from pccl_b200.models import SparseMoEBlock
    block = SparseMoEBlock(16, 32, 4, 2, dtype=torch.float64, device="cpu")
    x = torch.randn(7, 16, dtype=torch.float64, requires_grad=True)
    out = block.experts(x, torch.tensor([0, 2, 2, 5, 5], dtype=torch.int32))
    for row, e in enumerate((0, 0, 2, 2, 2)):
        gate, up = (block.w13[e] @ x[row]).chunk(2)
        torch.testing.assert_close(out[row], block.w2[e] @ (torch.nn.functional.silu(gate) * up))
    assert bool((out[5:] == 0).all())
    out.sum().backward()
    assert bool((block.w13.grad[[1, 3]] == 0).all()) and bool((block.w2.grad[[0, 2]] != 0).any()) and bool((x.grad[5:] == 0).all())


@pytest.mark.parametrize("tokens,text", [(2 ** 31 - 100, "2\\^31"), (2 ** 31 - 2 ** 16, "2\\^31"), (2 ** 31 - 2 ** 16 - 1, "CUDA device"),
                                         (2 ** 33, "2\\^31")])
def test_most_tokens_of_a_routing(tokens, text):
    """Token numbers and a block's tokens on top of them are 31-bit sums in the kernels."""
    with pytest.raises(ValueError, match=text):
        route_topk(torch.zeros(1, 1).expand(tokens, 1), 1)


def test_a_routing_of_one_allocation_is_pickled():
    """Its parts as route_topk makes them: whole numbers and weights in one storage, which torch.save refuses to write."""
    import copy
    import io
    all_ = torch.arange(100, dtype=torch.int32)
    r = Routing(all_[:8].view(4, 2), all_.view(torch.float32)[8:16].view(4, 2), all_[16:24].view(4, 2), all_[24:33])
    file = io.BytesIO()
    torch.save({"layer": r}, file)
    file.seek(0)
    for copied in (torch.load(file, weights_only=False)["layer"], copy.deepcopy(r), r._replace(rows=r.rows)):
        assert type(copied) is Routing and all(torch.equal(a, b) for a, b in zip(copied, r))


@pytest.mark.parametrize("grad", [False, True])
def test_rms_norm_needs_its_gamma(grad):
    """It returned None."""
    with pytest.raises(ValueError, match="rms_norm: gamma"):
        rms_norm(torch.zeros(4, 16, requires_grad=grad), None)
