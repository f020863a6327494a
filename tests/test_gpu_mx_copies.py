"""Copies of operands and plans stand on their own, and a question about a workspace changes no later call."""

import copy
import io
import pickle

import pytest
import torch

from comp_b200 import experts, mx

pytestmark = pytest.mark.gpu


def _saved(t):
    f = io.BytesIO()
    torch.save(t, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


COPIES = [copy.copy, copy.deepcopy, lambda t: pickle.loads(pickle.dumps(t)), _saved]


@pytest.mark.parametrize("of", COPIES)
def test_operand(cuda, of):
    x, w = torch.randn((3, 288), device=cuda), mx.quantize(torch.randn((130, 288), device=cuda))
    c = of(w)
    assert c.shape == w.shape and c.nbytes == w.nbytes and c._at == c.image.data_ptr() and c._index == w._index
    want, values = mx.linear(x, w), mx.dequantize(w)
    if of is not copy.copy:  # (whose image is the same one)
        assert c.image.data_ptr() != w.image.data_ptr()
        w.image.zero_()
    assert torch.equal(mx.linear(x, c), want) and torch.equal(mx.dequantize(c), values)
    many = mx.quantize(torch.randn((3, 40, 64), device=cuda))
    assert of(many).shape == (3, 40, 64)
    with pytest.raises(AttributeError):
        w.image = c.image


@pytest.mark.parametrize("of", COPIES)
@pytest.mark.parametrize("tokens", [5, 400])
def test_plan(cuda, of, tokens):
    w = mx.quantize(torch.randn((6, 40, 64), device=cuda))
    x, logits = torch.randn((tokens, 64), device=cuda), torch.randn((tokens, 6), device=cuda)
    routed = experts.route(logits, 3)
    ids, weights = routed.ids.clone(), routed.weights.clone()
    for plan in (routed, experts.sort(ids, 6)):
        c = of(plan)
        want = experts.combine(experts.linear(x, w, plan), plan, weights)
        pos = plan.pos.clone()
        if of is not copy.copy:
            assert c._at != plan._at
            plan._words.zero_()
        assert c._at == c.offsets.data_ptr() and torch.equal(c.pos, pos) and torch.equal(c.ids, ids)
        assert torch.equal(experts.combine(experts.linear(x, w, c), c, weights), want)
        if plan is routed:
            assert torch.equal(c.weights, weights)
        else:
            assert c.weights is None


def test_plan_of_another_layer(cuda):
    """A workspace's size is asked for with a plan of more experts than the weights have, which is refused; the next product is
    the right one."""
    w = mx.quantize(torch.randn((2, 300, 64), device=cuda))
    x = torch.randn((4, 64), device=cuda)
    other, plan = (experts.sort(torch.zeros((4, 1), dtype=torch.int32, device=cuda), n) for n in (300, 2))
    with pytest.raises(ValueError, match="expected"):
        experts.workspace_size(other, w)
    with pytest.raises(TypeError, match="Plan"):
        experts.workspace_size(None, w)
    with pytest.raises(TypeError, match="MXTensor"):
        experts.workspace_size(plan, None)
    assert torch.isfinite(experts.linear(x, w, plan)).all()
