"""A side without tokens beside documents, coordinates or both: an empty tensor has no address, and is given all the same."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("L,M", [(0, 5), (5, 0), (0, 0), (0, 700), (700, 0)])
@pytest.mark.parametrize("docs", [None, torch.int32, torch.int64])
@pytest.mark.parametrize("coords", [False, True])
def test_no_rows_or_no_keys(device, L, M, docs, coords):
    from dgl_amd.attention import attention, attention_backward, attention_forward
    g = torch.Generator(device=device).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    q, k, v, do = rnd(2, 4, L, 16), rnd(2, 2, M, 16), rnd(2, 2, M, 16), rnd(2, 4, L, 16)
    kw = {}
    if docs is not None:
        kw["doc_q"], kw["doc_k"] = (torch.zeros(2, n, dtype=docs, device=device) for n in (L, M))
    if coords:
        kw["slope"], kw["pos_q"], kw["pos_k"] = torch.rand(4, device=device), rnd(2, L, 2), rnd(2, M, 2)
    out, lse = attention_forward(q, k, v, **kw)
    assert out.shape == q.shape and not out.any() and torch.isneginf(lse).all()
    dq, dk, dv, ds = attention_backward(do, q, k, v, out, lse, **kw)
    assert dq.shape == q.shape and dk.shape == dv.shape == k.shape
    assert not dq.any() and not dk.any() and not dv.any() and (ds is None or not ds.any())
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    attention(*leaves, **kw).backward(do)
    for t in leaves:
        assert t.grad.shape == t.shape and not t.grad.any()
