"""A pool of pages that sequences share: which sequences there are, and what counts as stored."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_sequences_out_of_range_are_refused(device):
    from dgl_amd.attention import PagedCache
    cache = PagedCache(3, 1, 16, 64, page_size=16, num_pages=6, device=device)
    cache.reserve(2, 20)
    x = torch.randn(3, 1, 20, 16, device=device)
    cache.append(x, x, counts=torch.tensor([0, 0, 20], device=device, dtype=torch.int32))
    table, lengths = cache.table.clone(), cache.lengths.clone()
    for sequence in (-1, -3, 3, 100):
        with pytest.raises(ValueError, match="sequence"):
            cache.release(sequence)
        with pytest.raises(ValueError, match="sequence"):
            cache.reserve(sequence, 33)
    assert torch.equal(cache.table, table) and torch.equal(cache.lengths, lengths)
    cache.release(2)
    assert cache.lengths.tolist() == [0, 0, 0] and int(cache.table[2].max()) == -1
    cache.reserve(0, 64)
    cache.reserve(1, 32)                                  # all six pages are free again


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 40, 700])
def test_tokens_that_found_no_page_do_not_count(device, dtype, T):
    """One workgroup a sequence, and many (700 tokens of 4 heads of 64): the length ends at the first token without a page, and a
    page that comes later is read from the first token that is then stored in it, not for what another sequence left there."""
    from attention_reference import assert_within, reference
    from dgl_amd.attention import PagedCache, attention_step
    H, D, page = 4, 64, 16
    per = (T + 47) // page
    cache = PagedCache(4, H, D, per * page, page_size=page, num_pages=3 * per, dtype=dtype, device=device)
    g = torch.Generator(device=device).manual_seed(T)
    rnd = lambda n: torch.randn(4, H, n, D, device=device, generator=g).to(dtype)  # noqa: E731
    for s in range(3):
        cache.reserve(s, per * page)
    cache.append(*[torch.full((4, H, per * page, D), 1e4, device=device, dtype=dtype) for _ in range(2)])     # somebody's tokens
    assert cache.lengths.tolist() == [per * page] * 3 + [0]
    for s in range(3):
        cache.release(s)
    cache.lengths.zero_()
    have = [T // 2 // page * page, T, 0, 0]
    for s in range(4):
        cache.reserve(s, have[s])
    k, v = rnd(T), rnd(T)
    cache.append(k, v)
    want = [min(T, (n + page - 1) // page * page) for n in have]
    assert cache.lengths.tolist() == want
    cache.append(k[:, :, :0], v[:, :, :0])
    assert cache.lengths.tolist() == want
    for s in (0, 2):
        cache.reserve(s, T + 1)
    more = rnd(1), rnd(1)
    cache.append(*more, counts=torch.tensor([1, 0, 1, 1], device=device, dtype=torch.int32))
    q = torch.randn(4, H, D, device=device, generator=g).to(dtype)
    out = attention_step(q, cache)
    for s in range(3):
        n = want[s]
        ks, vs = (torch.cat((x[s:s + 1, :, :n], y[s:s + 1]), 2) if s != 1 else x[s:s + 1, :, :n] for x, y in zip((k, v), more))
        ref = reference(q[s:s + 1, :, None], ks, vs)["out"]
        assert_within(out[s:s + 1, :, None], ref, f"sequence {s}")
    assert int(cache.lengths[3]) == 0 and not out[3].any()


def test_pages_given_up_in_front_do_not_stop_a_sequence(device):
    """A window that slides: early pages absent, tokens go on behind them."""
    from dgl_amd.attention import PagedCache
    cache = PagedCache(1, 1, 16, 64, page_size=16, device=device)
    x = torch.randn(1, 1, 30, 16, device=device)
    cache.append(x, x)
    cache.table[0, 0] = -1
    cache.append(x[:, :, :20], x[:, :, :20])
    assert int(cache.lengths[0]) == 50
    cache.table[0, 3] = 10 ** 6
    cache.append(x, x)
    assert int(cache.lengths[0]) == 50
