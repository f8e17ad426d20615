"""Attention of one new token per row over the paged cache, and the cache's append, against the definition in 64 bits."""
import math

import pytest
import torch

from attention_reference import assert_within, reference

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make(B, P, H, K, D, lengths, page, dtype, seed, device="cuda", max_pages=None):
    """A cache with scattered pages; what lies behind a sequence's last token is NaN."""
    from dgl_amd.attention import PagedCache
    g = torch.Generator(device=device).manual_seed(seed)
    lengths = torch.tensor(lengths, device=device, dtype=torch.int32)
    n = max(1, int(lengths.max()))
    per = max_pages or (n + page - 1) // page
    total = B * per + 2
    kp = torch.full((total, K, page, D), math.nan, device=device, dtype=dtype)
    vp = kp.clone()
    table = torch.randperm(total, device=device, generator=g)[:B * per].view(B, per).to(torch.int32)
    k = torch.randn(B, K, per * page, D, device=device, generator=g).to(dtype)
    v = torch.randn(B, K, per * page, D, device=device, generator=g).to(dtype)
    for b in range(B):
        for j in range(int(lengths[b])):
            kp[table[b, j // page], :, j % page], vp[table[b, j // page], :, j % page] = k[b, :, j], v[b, :, j]
    q = torch.randn(B * P, H, D, device=device, generator=g).to(dtype)
    return PagedCache.over(kp, vp, table, lengths), q, k, v, g


def expected(q, k, v, lengths, P, scale=None, cap=0.0, slope=None, pos_q=None, pos_k=None, blocked=None, absent=None):
    R, H, D = q.shape
    n = k.shape[2]
    j = torch.arange(n, device=q.device)
    seq = torch.arange(R, device=q.device) // P
    seen = j[None] < lengths[seq][:, None]
    if blocked is not None:
        bits = (((blocked[:, :, None] >> torch.arange(64, device=q.device)) & 1) != 0).view(R, -1)[:, :n]
        seen = seen & ~torch.nn.functional.pad(bits, (0, n - bits.shape[1]))
    if absent is not None:
        seen = seen & ~absent[seq]
    if slope is not None and pos_q is None:      # the distance to the last live token, as coordinates on a line
        pos_q = torch.stack((lengths[seq].float() - 1, torch.zeros(R, device=q.device)), 1)
        pos_k = torch.stack((j.float(), torch.zeros(n, device=q.device)), 1).expand(k.shape[0], n, 2)
    if pos_k is not None and pos_k.shape[1] < n:
        pos_k = torch.nn.functional.pad(pos_k, (0, 0, 0, n - pos_k.shape[1]))
    kw = {} if slope is None else {"slope": slope, "pos_q": pos_q[:, None], "pos_k": pos_k[seq]}
    want = reference(q[:, :, None], k[seq], v[seq], scale=scale, cap=cap, doc_q=torch.zeros(R, 1, device=q.device, dtype=torch.int32),
                     doc_k=torch.where(seen, 0, -1).to(torch.int32), **kw)
    return tuple(x[:, :, 0] for x in want["out"]), tuple(x[:, :, 0] for x in want["lse"])


def check(cache, q, k, v, P, **kw):
    from dgl_amd.attention import attention_step
    absent = kw.pop("absent", None)
    out, lse = attention_step(q, cache, rows_per_instance=P, return_lse=True, **kw)
    want, want_lse = expected(q, k, v, cache.lengths, P, absent=absent, **kw)
    assert_within(out, want, "out")
    assert_within(lse, want_lse, "lse")
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [8, 16, 24, 32, 64, 72, 128])
@pytest.mark.parametrize("P,G", [(1, 1), (1, 8), (20, 1), (3, 16), (70, 1)])
def test_head_sizes_and_query_counts(device, dtype, D, P, G):
    cache, q, k, v, g = make(2, P, 2 * G, 2, D, [77, 40], 16, TYPES[dtype], D + P + G)
    check(cache, q, k, v, P)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("lengths", [[1, 0, 5], [31, 32, 33], [64, 63, 65], [300, 1, 257]])
def test_lengths_and_pages(device, dtype, page, lengths):
    cache, q, k, v, g = make(3, 2, 4, 2, 16, lengths, page, TYPES[dtype], page + sum(lengths))
    out = check(cache, q, k, v, 2, cap=5.0)
    for b, n in enumerate(lengths):
        if n == 0:
            assert not out[2 * b:2 * b + 2].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", ["index", "coords"])
@pytest.mark.parametrize("P", [1, 17, 50])
def test_bias_cap_and_blocked_bits(device, dtype, bias, P):
    cache, q, k, v, g = make(3, P, 4, 4, 16, [130, 97, 64], 32, TYPES[dtype], P)
    kw = {"cap": 4.0, "slope": torch.rand(4, device=device, generator=g) * (2.0 if bias == "coords" else 0.05)}
    if bias == "coords":
        kw["pos_q"] = torch.rand(3 * P, 2, device=device, generator=g)
        kw["pos_k"] = torch.rand(3, 131, 2, device=device, generator=g)
    bits = torch.randint(-2 ** 62, 2 ** 62, (3 * P, 2), device=device, generator=g)   # fewer words than tokens: the rest is seen
    bits[0] = -1
    kw["blocked"] = bits
    check(cache, q, k, v, P, **kw)
    kw["blocked"] = torch.full((3 * P, 3), -1, device=device)
    assert not check(cache, q, k, v, P, **kw).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("P,G,D", [(1, 1, 16), (1, 4, 128), (2, 4, 64), (20, 1, 16)])
def test_long_caches_are_split_and_joined(device, dtype, P, G, D):
    from dgl_amd import _lib
    cache, q, k, v, g = make(2, P, G, 1, D, [5000, 33], 64, TYPES[dtype], D)
    a = _lib.AttentionStep()
    a.cache, a.rows_per_instance, a.Hq, a.scale = cache.struct, P, G, 1.0
    a.q = a.out = 4096
    import ctypes
    assert _lib.load().dgl_attention_step_workspace_floats(ctypes.byref(a)) > 0
    check(cache, q, k, v, P, cap=20.0, slope=torch.full((G,), 0.01, device=device))
    blocked = torch.zeros(2 * P, 79, dtype=torch.int64, device=device)
    blocked[:, 3:70] = -1                        # whole ranges of the split see nothing
    check(cache, q, k, v, P, blocked=blocked)


@pytest.mark.parametrize("dtype", TYPES)
def test_absent_pages_and_lengths_out_of_range(device, dtype):
    cache, q, k, v, g = make(3, 2, 2, 2, 32, [100, 128, 90], 32, TYPES[dtype], 1)
    absent = torch.zeros(3, 128, dtype=torch.bool, device=device)
    cache.table[0, 1], absent[0, 32:64] = -1, True
    cache.table[1, 2], absent[1, 64:96] = 10 ** 9, True
    check(cache, q, k, v, 2, absent=absent)
    cache.lengths[1], cache.lengths[2] = 10 ** 9, -5     # as many as the table holds; none
    from dgl_amd.attention import attention_step
    out = attention_step(q, cache, rows_per_instance=2)
    want, _ = expected(q, k, v, torch.tensor([100, 128, 0], device=device), 2, absent=absent)
    assert_within(out, want, "out")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [90, 3000])
def test_blocked_keys_hold_anything(device, dtype, n):
    from dgl_amd.attention import attention_step
    cache, q, k, v, g = make(1, 3, 2, 1, 16, [n], 32, TYPES[dtype], 3)
    blocked = torch.zeros(3, (n + 63) // 64, dtype=torch.int64, device=device)
    blocked[:2, 0] = 1 << 7                      # key 7 is blocked for rows 0 and 1
    page, slot = int(cache.table[0, 0]), 7
    cache.v_pages[page, :, slot] = math.nan
    cache.k_pages[page, :, slot] = math.inf
    out = attention_step(q, cache, rows_per_instance=3, blocked=blocked)
    want, _ = expected(q[:2], torch.where(torch.isfinite(k), k, 0), v, cache.lengths, 2, blocked=blocked[:2])
    k0, v0 = k.clone(), v.clone()
    assert_within(out[:2], want, "rows that do not see the poisoned key")
    assert out[2].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_append_writes_tokens_and_nothing_else(device, dtype):
    from dgl_amd.attention import PagedCache
    t = TYPES[dtype]
    cache = PagedCache(3, 2, 16, 100, page_size=16, dtype=t, device=device)
    cache.k_pages.fill_(7.0)
    cache.v_pages.fill_(-7.0)
    g = torch.Generator(device=device).manual_seed(0)
    ref_k = torch.full((3, 2, 112, 16), 7.0, device=device, dtype=t)
    ref_v = torch.full((3, 2, 112, 16), -7.0, device=device, dtype=t)
    lengths = [0, 0, 0]

    def put(T, counts=None, start=None):
        k = torch.randn(3, T, 2, 16, device=device, generator=g).to(t).transpose(1, 2)
        v = torch.randn(3, 2, T, 16, device=device, generator=g).to(t)
        c = None if counts is None else torch.tensor(counts, device=device, dtype=torch.int32)
        s = None if start is None else torch.tensor(start, device=device, dtype=torch.int32)
        cache.append(k, v, counts=c, start=s)
        for b in range(3):
            first = lengths[b] if start is None else start[b]
            m = T if counts is None else min(max(counts[b], 0), T)
            for x in range(m):
                if 0 <= first + x < 112:
                    ref_k[b, :, first + x], ref_v[b, :, first + x] = k[b, :, x], v[b, :, x]
            lengths[b] = min(max(first + m, 0), 112)
        rows = cache.table.long()
        assert cache.lengths.tolist() == lengths
        assert torch.equal(cache.k_pages[rows].transpose(1, 2).reshape(3, 2, 112, 16), ref_k)
        assert torch.equal(cache.v_pages[rows].transpose(1, 2).reshape(3, 2, 112, 16), ref_v)
    put(37, counts=[37, 0, 20])                  # a ragged prompt
    put(1)
    put(1, counts=[1, 1, 0])
    put(1, start=[5, 0, 100])
    put(60, counts=[99, -3, 60])                 # counts beyond the batch's tokens, below zero; past the capacity
    put(3, start=[-1, 110, 200])


def test_long_prompt_takes_many_workgroups(device):
    from dgl_amd.attention import PagedCache
    cache = PagedCache(2, 4, 64, 3000, page_size=64, device=device)
    k, v = torch.randn(2, 2, 4, 2500, 64, device=device).unbind(0)
    counts = torch.tensor([2500, 1234], device=device, dtype=torch.int32)
    cache.append(k, v, counts=counts)
    assert cache.lengths.tolist() == [2500, 1234]
    got = cache.k_pages[cache.table.long()].transpose(1, 2).reshape(2, 4, -1, 64)
    assert torch.equal(got[0, :, :2500], k[0]) and torch.equal(got[1, :, :1234], k[1, :, :1234])
    assert not got[1, :, 1234:].any()


def test_pool_of_pages(device):
    from dgl_amd.attention import PagedCache, attention_step
    cache = PagedCache(3, 1, 16, 64, page_size=16, num_pages=6, device=device)
    cache.reserve(0, 40)
    cache.reserve(2, 17)
    with pytest.raises(RuntimeError, match="free"):
        cache.reserve(1, 32)
    with pytest.raises(ValueError, match="at most"):
        cache.reserve(1, 65)
    x = torch.randn(3, 1, 17, 16, device=device)
    cache.append(x, x)                           # sequence 1 has no page: its tokens are dropped
    q = torch.randn(3, 1, 16, device=device)
    out = attention_step(q, cache)
    assert not out[1].any() and out[0].any() and out[2].any()
    pages = set(cache.table[0, :3].tolist()) | set(cache.table[2, :2].tolist())
    assert len(pages) == 5
    cache.release(0)
    cache.reserve(1, 64)
    assert cache.lengths[0] == 0 and not attention_step(q, cache)[0].any()
    torch.testing.assert_close(attention_step(q, cache)[2], out[2], rtol=0, atol=0)


def test_a_rollout_of_appends_and_steps_equals_one_causal_pass(device):
    """Prompt, then token by token: the steps together are the causal operator with the positions' bias."""
    from dgl_amd.attention import PagedCache, attention_forward, attention_step
    B, H, K, D, n, prompt = 2, 4, 2, 16, 70, 33
    g = torch.Generator(device=device).manual_seed(5)
    q = torch.randn(B, H, n, D, device=device, generator=g)
    k, v = (torch.randn(B, K, n, D, device=device, generator=g) for _ in range(2))
    slope = torch.tensor([0.1, 0.2, 0.05, 0.0], device=device)
    whole, _ = attention_forward(q, k, v, causal=True, cap=6.0, slope=slope)
    want = reference(q, k, v, causal=True, cap=6.0, slope=slope)["out"]
    cache = PagedCache(B, K, D, n, page_size=16, device=device)
    cache.append(k[:, :, :prompt], v[:, :, :prompt])
    for t in range(prompt, n):
        cache.append(k[:, :, t:t + 1], v[:, :, t:t + 1])
        step = attention_step(q[:, :, t].contiguous(), cache, cap=6.0, slope=slope)
        assert_within(step, (want[0][:, :, t], want[1][:, :, t]), f"step {t}")
    assert_within(whole, want, "whole")


def test_captured_step_follows_lengths_and_bits(device):
    from dgl_amd.attention import PagedCache, attention_step
    cache = PagedCache(2, 2, 16, 4096, page_size=64, device=device)
    x = torch.randn(2, 2, 2, 4096, 16, device=device)
    cache.append(x[0][:, :, :4000], x[1][:, :, :4000])
    q = torch.randn(6, 2, 16, device=device)
    new = torch.randn(2, 2, 2, 1, 16, device=device)
    blocked = torch.zeros(6, 64, dtype=torch.int64, device=device)

    def one():
        cache.append(new[0], new[1])
        return attention_step(q, cache, rows_per_instance=3, blocked=blocked)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        one()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = one()
    assert cache.lengths.tolist() == [4001, 4001]        # a capture runs nothing
    for i in range(3):
        blocked[:, i] = -1
        q.add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert cache.lengths.tolist() == [4002 + i] * 2
        assert torch.equal(out, attention_step(q, cache, rows_per_instance=3, blocked=blocked))


def test_strided_queries_pages_and_other_streams(device):
    from dgl_amd.attention import PagedCache, attention_step
    g = torch.Generator(device=device).manual_seed(3)
    kv = torch.randn(9, 32, 2, 2, 16, device=device, generator=g)        # [page, slot, k/v, head, size]
    table = torch.arange(8, device=device, dtype=torch.int32).view(2, 4)
    lengths = torch.tensor([100, 128], device=device, dtype=torch.int32)
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    cache = PagedCache.over(k, v, table, lengths)
    dense = PagedCache.over(k.contiguous(), v.contiguous(), table, lengths)
    x = torch.randn(2, 6, 3, 16, device=device, generator=g)
    q = x[:, :, 1]
    a = attention_step(q, cache)
    assert torch.equal(a, attention_step(q.contiguous(), dense))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = attention_step(q, cache)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, b)


def test_refusals(device):
    from dgl_amd.attention import PagedCache, attention_step
    cache = PagedCache(2, 2, 16, 64, device=device)
    q = torch.randn(2, 4, 16, device=device)
    for bad in (q[0], q[:1], q[:, :3], q[:, :, :8], q.half(), q.cpu()):
        with pytest.raises(ValueError):
            attention_step(bad, cache)
    with pytest.raises(ValueError):
        attention_step(q, cache, pos_q=torch.zeros(2, 2, device=device), pos_k=torch.zeros(2, 64, 2, device=device))
    with pytest.raises(ValueError):
        attention_step(q, cache, blocked=torch.zeros(2, 1, device=device))
    with pytest.raises(ValueError):
        cache.append(torch.zeros(2, 2, 1, 8, device=device), torch.zeros(2, 2, 1, 8, device=device))
    with pytest.raises(ValueError):
        PagedCache.over(cache.k_pages, cache.v_pages, cache.table.long(), cache.lengths)
