"""Refusals of routing, dispatch / combine and the block norms: every check runs before anything touches a GPU."""

import pytest
import torch

from pccl_b200.ops import Routing, combine, dispatch, residual_rms_norm, rms_norm, route_topk


def _routing(t=4, k=2, e=8, **change):
    parts = dict(idx=torch.zeros(t, k, dtype=torch.int32), weights=torch.zeros(t, k), offsets=torch.zeros(e + 1, dtype=torch.int32),
                 rows=torch.arange(t * k, dtype=torch.int32).view(t, k))
    return Routing(**{**parts, **change})


@pytest.mark.parametrize("change,text", [
    (dict(logits=torch.zeros(4)), "tokens, experts"),
    (dict(logits=torch.zeros(4, 8, dtype=torch.float64)), "float32, float16 or bfloat16"),
    (dict(logits=torch.zeros(4, 0)), "1 to 1024 experts"),
    (dict(logits=torch.zeros(1, 1025)), "1 to 1024 experts"),
    (dict(top_k=0), "top_k"),
    (dict(top_k=9), "top_k"),
    (dict(logits=torch.zeros(1, 64), top_k=32), "top_k"),
    (dict(groups=3), "groups"),
    (dict(logits=torch.zeros(1, 66), groups=33), "groups"),
    (dict(groups=0), "groups"),
    (dict(groups=4, top_groups=5), "top_groups"),
    (dict(groups=4, top_groups=0), "top_groups"),
    (dict(groups=4, top_groups=1, top_k=3), "top_k"),
    (dict(groups=8, top_groups=2, group_score="top2"), "groups of two"),
    (dict(scoring="tanh"), "scoring"),
    (dict(group_score="mean"), "group_score"),
    (dict(bias=torch.zeros(7)), "bias"),
    (dict(bias=torch.zeros(8, dtype=torch.bfloat16)), "bias"),
    (dict(bias=torch.zeros(8, requires_grad=True)), "no gradient"),
    (dict(mask=torch.ones(4)), "mask"),
    (dict(mask=torch.ones(3, dtype=torch.bool)), "mask"),
    (dict(), "CUDA device"),
])
def test_route_topk_refuses(change, text):
    args = {**dict(logits=torch.zeros(4, 8), top_k=2), **change}
    with pytest.raises(ValueError, match=text):
        route_topk(args.pop("logits"), args.pop("top_k"), **args)


@pytest.mark.parametrize("op", [dispatch, combine])
@pytest.mark.parametrize("change,text", [
    (dict(x=torch.zeros(8)), "matrix"),
    (dict(x=torch.zeros(8, 16, dtype=torch.int32)), "matrix"),
    (dict(x=torch.zeros(8, 0)), "at least one value"),
    (dict(x=torch.zeros(7, 16)), "rows"),
    (dict(rows=torch.zeros(4, 2, dtype=torch.int64)), "routing.rows"),
    (dict(rows=torch.zeros(2, 4, dtype=torch.int32).t()), "routing.rows"),
    (dict(rows=torch.zeros(4, 0, dtype=torch.int32)), "top_k"),
    (dict(offsets=torch.zeros(9)), "routing.offsets"),
    (dict(offsets=torch.zeros(0, dtype=torch.int32)), "routing.offsets"),
    (dict(), "CUDA device"),
])
def test_moves_refuse(op, change, text):
    x = change.get("x", torch.zeros(4 if op is dispatch else 8, 16))
    with pytest.raises(ValueError, match=text):
        op(x, _routing(**{n: v for n, v in change.items() if n != "x"}))


@pytest.mark.parametrize("weights", [torch.zeros(4, 2, dtype=torch.float64), torch.zeros(4, 3), torch.zeros(2, 4).t()])
def test_combine_refuses_other_weights(weights):
    with pytest.raises(ValueError, match="routing.weights"):
        combine(torch.zeros(8, 16), _routing(weights=weights))


@pytest.mark.parametrize("change,text", [
    (dict(residual=torch.zeros(())), "hidden"),
    (dict(residual=torch.zeros(4, 16, dtype=torch.float64)), "float32, float16 or bfloat16"),
    (dict(x=torch.zeros(4, 16, dtype=torch.int8)), "float32, float16 or bfloat16"),
    (dict(residual=torch.zeros(4, 0), x=torch.zeros(4, 0)), "hidden must be between"),
    (dict(residual=torch.zeros(1, 16385), x=torch.zeros(1, 16385)), "hidden must be between"),
    (dict(x=torch.zeros(16, 4)), "same shape"),
    (dict(residual=torch.zeros(4, 16, dtype=torch.bfloat16)), "type of x or float32"),
    (dict(gamma=torch.zeros(15)), "gamma"),
    (dict(gamma=torch.zeros(1, 16)), "gamma"),
    (dict(gamma=torch.zeros(16, dtype=torch.float16)), "gamma"),
    (dict(post_gamma=torch.zeros(17)), "post_gamma"),
    (dict(gate=torch.zeros(3, 16)), "divide evenly"),
    (dict(gate=torch.zeros(0, 16)), "divide evenly"),
    (dict(gate=torch.zeros(2, 2, 16)), "gate"),
    (dict(gate=torch.zeros(16, dtype=torch.bfloat16)), "gate"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(x=None), "rms_norm"),
    (dict(), "CUDA device"),
])
def test_residual_rms_norm_refuses(change, text):
    args = {**dict(residual=torch.zeros(4, 16), x=torch.zeros(4, 16), gamma=torch.ones(16)), **change}
    with pytest.raises(ValueError, match=text):
        residual_rms_norm(args.pop("residual"), args.pop("x"), args.pop("gamma"), **args)


def test_rms_norm_refuses():
    with pytest.raises(ValueError, match="gamma"):
        rms_norm(torch.zeros(4, 16, dtype=torch.bfloat16), torch.ones(16, dtype=torch.float16))
    with pytest.raises(ValueError, match="CUDA device"):
        rms_norm(torch.zeros(4, 16), torch.ones(16))
