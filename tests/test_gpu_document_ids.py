"""Document ids are whole numbers of any integer type: those beyond 32 bits keep what they tell apart."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def run(q, k, v, do, doc_q, doc_k, **kw):
    from dgl_amd.attention import attention_backward, attention_forward
    out, lse = attention_forward(q, k, v, doc_q=doc_q, doc_k=doc_k, **kw)
    return (out, lse) + attention_backward(do, q, k, v, out, lse, doc_q=doc_q, doc_k=doc_k, **kw)[:3]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def tensors(B, H, L, M, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda n: torch.randn(B, H, n, 16, device=device, generator=g)  # noqa: E731
    return rnd(L), rnd(M), rnd(M), rnd(L)


@pytest.mark.parametrize("base", [0, 2 ** 31 - 2, 2 ** 31, 2 ** 40 + 5, 2 ** 63 - 5])
@pytest.mark.parametrize("causal", [False, True])
def test_neighbouring_wide_ids_are_different_documents(device, base, causal):
    t = tensors(2, 2, 150, 150, device)
    small = torch.sort(torch.randint(0, 4, (2, 150), device=device), 1)[0]
    small[1, -9:] = -3
    wide = torch.where(small < 0, small - 2 ** 50, small + base)
    assert same(run(*t, wide, wide, causal=causal), run(*t, small.int(), small.int(), causal=causal))


def test_ids_in_any_order_with_equal_low_halves(device):
    """Ids that agree in their lower 32 bits, in no order, another set on either side; rows of ids that no key has."""
    t = tensors(3, 2, 130, 333, device, 1)
    g = torch.Generator(device=device).manual_seed(3)
    i, j = torch.randint(0, 20, (3, 130), device=device, generator=g), torch.randint(0, 15, (3, 333), device=device, generator=g)
    i[:, 50], j[:, 7] = -1, -1
    far = lambda x: torch.where(x < 0, x, x * 2 ** 32 + 77)  # noqa: E731
    assert same(run(*t, far(i), far(j)), run(*t, i.int(), j.int()))
    assert same(run(*t, i.int(), j), run(*t, i.int(), j.int()))            # types of the two sides may differ


def test_many_documents(device):
    """Every token its own document but for the pairs that an offset makes: 20 000 keys."""
    t = tensors(1, 1, 20000, 20000, device, 2)
    ids = torch.randperm(20000, device=device, generator=torch.Generator(device=device).manual_seed(4))[None] // 2
    wide = ids * 2 ** 33 + 2 ** 45
    assert same(run(*t, wide, wide), run(*t, ids.int(), ids.int()))


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.bool, torch.uint16, torch.uint32])
def test_other_integer_types(device, dtype):
    t = tensors(1, 2, 60, 60, device, 3)
    ids = (torch.arange(60, device=device) >= 25).int()[None]
    top = {torch.uint8: 254, torch.uint16: 2 ** 16 - 2, torch.uint32: 2 ** 32 - 2}.get(dtype, 0)
    narrow = (ids.to(torch.int64) + top).to(dtype)
    assert same(run(*t, narrow, narrow), run(*t, ids, ids))


def test_broadcast_and_strided_ids(device):
    t = tensors(4, 1, 90, 90, device, 4)
    one = (torch.arange(90, device=device) // 40 + 2 ** 36)[None]
    ids = (torch.arange(90, device=device, dtype=torch.int32) // 40).expand(4, 90).contiguous()
    assert same(run(*t, one.expand(4, 90), one.expand(4, 90)), run(*t, ids, ids))
    apart = torch.stack((one.expand(4, 90), torch.full((4, 90), 3, device=device)), -1)[..., 0]
    assert same(run(*t, apart, apart), run(*t, ids, ids))


def test_refusals(device):
    from dgl_amd.attention import attention
    q = torch.zeros(1, 1, 8, 16, device=device)
    ids = torch.zeros(1, 8, dtype=torch.int64, device=device)
    for bad in (ids.float(), ids[:, :7], ids.cpu(), ids.to(torch.uint64)):
        with pytest.raises(ValueError, match="doc_q"):
            attention(q, q, q, doc_q=bad, doc_k=ids)
        with pytest.raises(ValueError, match="doc_k"):
            attention(q, q, q, doc_q=ids, doc_k=bad)


def test_captured_call_follows_the_ids(device):
    from dgl_amd.attention import attention_forward
    q, k, v, _ = tensors(2, 2, 100, 100, device, 6)
    ids = torch.zeros(2, 100, dtype=torch.int64, device=device)
    call = lambda: attention_forward(q, k, v, doc_q=ids, doc_k=ids)[0]  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        ids.copy_((torch.arange(100, device=device) // (20 + 9 * i))[None] * 2 ** (30 + i) - int(i == 2))
        graph.replay()
        torch.cuda.synchronize()
        narrow = torch.unique(ids, return_inverse=True)[1].int()
        narrow = torch.where(ids < 0, -1, narrow).to(torch.int32)
        assert torch.equal(out, attention_forward(q, k, v, doc_q=narrow, doc_k=narrow)[0]) and torch.equal(out, call())
