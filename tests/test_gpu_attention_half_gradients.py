"""Score gradients in half precision are scaled into its range by the rows' own size: rows that give no gradient (padding,
tokens outside a loss, rows without a key) leave that scale to the others."""
import math

import pytest
import torch

from attention_reference import assert_within, reference

pytestmark = pytest.mark.gpu


def inputs(H, K, L, M, D, seed, grad, device):
    """Large queries against small keys: dk = scale du^T q lies well above the spacing of half precision (2^-24), so that the
    rounding of du shows and not that of the stored gradient."""
    g = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    q, k = (64 * rnd(1, H, L, D)).half(), (rnd(1, K, M, D) / 64).half()
    return q, k, rnd(1, K, M, D).half(), (grad * rnd(1, H, L, D)).half()


def check(q, k, v, do, seen=None, **kw):
    """Gradients of both ways to drive the backward pass, against the definition for the rows in `seen`."""
    from dgl_amd.attention import attention, attention_backward, attention_forward
    out, lse = attention_forward(q, k, v, **kw)
    pair = attention_backward(do, q, k, v, out, lse, **kw)[:3]
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    attention(*leaves, **kw).backward(do)
    want = reference(q, k, v, do.nan_to_num(0.0, 0.0, 0.0), **kw)
    for got in (pair, [t.grad for t in leaves]):
        for x, n in zip(got, ("dq", "dk", "dv")):
            part = slice(None) if seen is None or n != "dq" else seen
            assert_within(x[:, :, part], tuple(y[:, :, part] for y in want[n]), n)
    return pair


@pytest.mark.parametrize("grad", [1e-4, 1e-6])
@pytest.mark.parametrize("H,K,L,M,D", [(2, 1, 100, 100, 16), (1, 1, 130, 70, 64), (2, 2, 96, 96, 128)])
@pytest.mark.parametrize("zero", ["none", "one", "most"])
def test_rows_without_a_gradient(device, grad, H, K, L, M, D, zero):
    q, k, v, do = inputs(H, K, L, M, D, 1, grad, device)
    if zero == "one":
        do[:, :, 17] = 0
    elif zero == "most":
        do[:, :, 10:] = 0
    check(q, k, v, do)


def test_a_gradient_of_zeros(device):
    q, k, v, do = inputs(2, 1, 90, 90, 32, 2, 1.0, device)
    for x in check(q, k, v, torch.zeros_like(do)):
        assert not x.any()


@pytest.mark.parametrize("fill", [0.0, 300.0, math.inf, math.nan])
def test_padding_rows(device, fill):
    """Padded tokens of packed documents, whose gradient may be anything."""
    q, k, v, do = inputs(2, 1, 200, 200, 32, 3, 1e-6, device)
    ids = (torch.arange(200, device=device) // 70).to(torch.int32)[None].clone()
    ids[:, 180:] = -1
    do[:, :, 180:] = fill
    check(q, k, v, do, doc_q=ids, doc_k=ids)


@pytest.mark.parametrize("fill", [0.0, 300.0, math.inf, math.nan])
def test_rows_that_see_no_key(device, fill):
    """Causal rows in front of the first key."""
    q, k, v, do = inputs(1, 1, 160, 60, 32, 4, 1e-6, device)
    do[:, :, :100] = fill
    check(q, k, v, do, causal=True)


def test_rows_with_a_single_key(device):
    """Documents of one token beside one of eighty: their score gradients are zero, whatever the size of their own gradient."""
    q, k, v, do = inputs(2, 1, 100, 100, 32, 6, 1e-6, device)
    ids = torch.arange(100, device=device, dtype=torch.int32).clamp_min(79)[None].clone()
    do[:, :, 80:] = (do[:, :, 80:].float() * 2e8).half()
    dk = check(q, k, v, do, doc_q=ids, doc_k=ids)[1]
    assert not dk[:, :, 80:].any()


def test_ranges_of_rows_and_heads(device):
    """Few keys against many rows: several workgroups share a block of keys, one range has gradients at all."""
    q, k, v, do = inputs(4, 1, 1100, 64, 32, 5, 1e-6, device)
    do[:, :, :1060] = 0
    do[:, 1] = 0
    check(q, k, v, do)
