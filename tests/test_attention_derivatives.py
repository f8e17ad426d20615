"""Gradients and tangents that a call would drop are refused before anything else is looked at (no GPU needed)."""
import pytest
import torch
from torch.autograd import forward_ad

from dgl_amd.attention import PagedCache, attention, attention_step
from dgl_amd.logits import process_logits


def leaf(*shape):
    return torch.zeros(*shape, requires_grad=True)


def calls():
    """(name of the input, call with it)"""
    q, x = torch.zeros(2, 4, 16), torch.zeros(1, 2, 4, 16)
    pos = torch.zeros(1, 4, 2)
    append = PagedCache.append
    return [
        ("q", lambda t: attention_step(t, None), q), ("slope", lambda t: attention_step(q, None, slope=t), torch.zeros(4)),
        ("pos_q", lambda t: attention_step(q, None, slope=torch.zeros(4), pos_q=t, pos_k=pos), torch.zeros(2, 2)),
        ("pos_k", lambda t: attention_step(q, None, slope=torch.zeros(4), pos_q=torch.zeros(2, 2), pos_k=t), pos),
        ("k_new", lambda t: append(None, t, x), x), ("v_new", lambda t: append(None, x, t), x),
        ("logits", lambda t: process_logits(t), torch.zeros(2, 5)), ("bias", lambda t: process_logits(torch.zeros(2, 5), bias=t), torch.zeros(5)),
        ("repetition", lambda t: process_logits(torch.zeros(2, 5), repetition=t), torch.ones(2)),
        ("presence", lambda t: process_logits(torch.zeros(2, 5), presence=t), torch.ones(2)),
        ("frequency", lambda t: process_logits(torch.zeros(2, 5), frequency=t), torch.ones(2)),
        ("pos_q", lambda t: attention(x, x, x, slope=torch.zeros(2), pos_q=t, pos_k=pos), pos),
        ("pos_k", lambda t: attention(x, x, x, slope=torch.zeros(2), pos_q=pos, pos_k=t), pos),
    ]


@pytest.mark.parametrize("at", range(13))
def test_gradients_are_refused_where_none_passes(at):
    name, call, value = calls()[at]
    with pytest.raises(ValueError, match=f"{name} requires grad"):
        call(value.clone().requires_grad_())
    with pytest.raises(ValueError, match=f"{name} requires grad"):
        call(value.clone().requires_grad_() * 1.0)               # not a leaf


@pytest.mark.parametrize("at", range(13))
def test_tangents_are_refused(at):
    name, call, value = calls()[at]
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match=f"{name} has a tangent"):
            call(forward_ad.make_dual(value, torch.ones_like(value)))


@pytest.mark.parametrize("at", range(4))
def test_attention_refuses_tangents_of_its_operands(at):
    t = [torch.zeros(1, 2, 4, 16) for _ in range(3)] + [torch.zeros(2)]
    for other in (False, True):                                  # beside an operand in reverse mode as well
        with forward_ad.dual_level():
            x = list(t)
            x[at] = forward_ad.make_dual(t[at], torch.ones_like(t[at]))
            if other:
                x[(at + 1) % 4] = t[(at + 1) % 4].clone().requires_grad_()
            with pytest.raises(ValueError, match="has a tangent"):
                attention(*x[:3], slope=x[3])


def test_without_gradients_the_calls_go_on():
    """Under no_grad the next check answers (these tensors are on the CPU, the cache is none)."""
    for name, call, value in calls():
        with torch.no_grad():
            with pytest.raises((ValueError, AttributeError)) as e:
                call(value.clone().requires_grad_())
        assert "requires grad" not in str(e.value)
