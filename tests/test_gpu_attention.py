"""The attention operator (dgl_amd/attention.py) against the definition in 64 bits: values and gradients for every
type, head layout, bias and mask, lengths from 0, strides, masked places holding NaN, refusals."""
import math

import pytest
import torch

from attention_reference import assert_within, reference

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def inputs(B, H, K, L, M, D, dtype, seed, bias="none", docs=0, prefix=False, device="cuda", grad=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    t = {"q": rnd(B, H, L, D).to(dtype), "k": rnd(B, K, M, D).to(dtype), "v": rnd(B, K, M, D).to(dtype),
         "dout": (grad * rnd(B, H, L, D)).to(dtype)}
    kw = {}
    if bias != "none":
        kw["slope"] = (0.3 + torch.rand(H, device=device, generator=g)) * (3.0 if bias == "coords" else 0.05)
    if bias == "coords":
        kw["pos_q"] = torch.rand(B, L, 2, device=device, generator=g)
        kw["pos_k"] = torch.rand(B, M, 2, device=device, generator=g)
    if docs:
        # ids in any order, padding on either side
        kw["doc_q"] = torch.randint(-1, docs, (B, L), device=device, generator=g).to(torch.int32)
        kw["doc_k"] = torch.randint(-1, docs, (B, M), device=device, generator=g).to(torch.int32)
    if prefix:
        kw["prefix"] = torch.randint(0, M + 1, (B,), device=device, generator=g).to(torch.int32)
    return t, kw


def check_all(t, kw, scale=None, cap=0.0, causal=False):
    from dgl_amd.attention import attention_backward, attention_forward
    kw = dict(kw, scale=scale, cap=cap, causal=causal)
    out, lse = attention_forward(t["q"], t["k"], t["v"], **kw)
    dq, dk, dv, dslope = attention_backward(t["dout"], t["q"], t["k"], t["v"], out, lse, **kw)
    got = {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    if dslope is not None:
        got["dslope"] = dslope
    want = reference(t["q"], t["k"], t["v"], t["dout"], **kw)
    for n in got:
        assert_within(got[n], want[n], n)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [8, 16, 24, 32, 64, 72, 128])
def test_head_sizes(device, dtype, D):
    t, kw = inputs(2, 2, 2, 70, 70, D, TYPES[dtype], D)
    check_all(t, kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L,M", [(1, 1), (1, 65), (17, 1), (63, 64), (64, 63), (65, 129), (130, 40), (200, 257)])
@pytest.mark.parametrize("bias,cap", [("none", 0.0), ("index", 10.0), ("coords", 3.0)])
def test_lengths_bias_cap(device, dtype, L, M, bias, cap):
    t, kw = inputs(2, 4, 2, L, M, 16, TYPES[dtype], L * 1000 + M, bias=bias)
    check_all(t, kw, cap=cap)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L,M", [(1, 1), (100, 100), (33, 161), (161, 33)])
@pytest.mark.parametrize("prefix", [False, True])
def test_causal_and_prefix(device, dtype, L, M, prefix):
    t, kw = inputs(3, 4, 1, L, M, 32, TYPES[dtype], L + M, bias="index", prefix=prefix)
    check_all(t, kw, causal=True)              # (161, 33): the first rows see nothing


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_documents_in_any_order_with_padding(device, dtype, causal):
    t, kw = inputs(3, 2, 1, 150, 150, 16, TYPES[dtype], 5, bias="coords", docs=3)
    kw["doc_q"][1] = -1                        # a row of padding only
    kw["doc_k"][2] = 7                         # documents that nobody asks for
    got = check_all(t, kw, cap=5.0, causal=causal)
    assert not got["out"][1].any() and torch.isneginf(got["lse"][1]).all() and not got["dk"][2].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_sorted_documents_skip_tiles(device, dtype):
    L = 700
    t, kw = inputs(2, 2, 2, L, L, 16, TYPES[dtype], 8)
    ids = torch.sort(torch.randint(0, 5, (2, L), device=device, generator=torch.Generator(device=device).manual_seed(1)), 1)[0]
    ids[:, 128:320] = ids[:, 128:129]          # whole tiles of one document
    ids = torch.sort(ids, 1)[0]
    ids[1, -30:] = -1
    kw["doc_q"] = kw["doc_k"] = ids.to(torch.int32)
    check_all(t, kw, causal=True)
    check_all(t, kw)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_take_two_blocks_per_wave(device, dtype):
    """From 512 workgroups of 128 rows on a wave holds two blocks of rows."""
    t, kw = inputs(32, 8, 8, 260, 260, 16, TYPES[dtype], 3, bias="coords")
    check_all(t, kw, cap=10.0)
    t, kw = inputs(32, 8, 8, 200, 260, 64, TYPES[dtype], 3, bias="index")
    check_all(t, kw, causal=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_two_blocks_wide_heads(device, dtype, D):
    t, kw = inputs(64, 8, 8, 70, 90, D, TYPES[dtype], 3)
    check_all(t, kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("H,K,L,M,D", [(2, 1, 5, 3000, 16), (8, 2, 600, 1100, 64), (4, 1, 1500, 130, 32), (8, 1, 1200, 1200, 128)])
def test_long_sides_are_split_and_joined(device, dtype, causal, H, K, L, M, D):
    """Few rows against many keys (forward), few keys or many shared heads against many rows (backward)."""
    t, kw = inputs(1, H, K, L, M, D, TYPES[dtype], L, bias="coords")
    kw["doc_q"] = torch.zeros(1, L, dtype=torch.int32, device=device)
    kw["doc_k"] = torch.zeros(1, M, dtype=torch.int32, device=device)
    kw["doc_k"][0, 100:120] = -1
    t["v"][:, :, 100:120] = math.nan
    check_all(t, kw, cap=8.0, causal=causal)


def test_scores_of_large_magnitude_and_flat_caps(device):
    t, kw = inputs(1, 2, 2, 80, 80, 16, torch.float32, 4)
    check_all({**t, "q": t["q"] * 30}, kw)                       # nearly one-hot rows
    check_all({**t, "q": t["q"] * 1000}, kw, cap=20.0)           # saturated tanh
    check_all(t, kw, cap=5000.0)                                 # tanh in its linear part
    check_all(t, kw, scale=-0.7)
    check_all(t, kw, scale=0.0)


@pytest.mark.parametrize("grad", [1e-6, 1.0, 300.0])
def test_half_precision_gradients_of_any_scale(device, grad):
    t, kw = inputs(1, 2, 1, 300, 300, 32, torch.float16, 6, grad=grad)
    check_all(t, kw)


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_and_broadcast_operands(device, dtype):
    from dgl_amd.attention import attention_forward
    t = TYPES[dtype]
    g = torch.Generator(device=device).manual_seed(9)
    x = torch.randn(2, 90, 3, 4, 16, device=device, generator=g).to(t)          # [batch, token, q/k/v, head, size]
    q, k, v = (x[:, :, i].transpose(1, 2) for i in range(3))
    dense = [u.contiguous() for u in (q, k, v)]
    dout = torch.randn(2, 4, 90, 16, device=device, generator=g).to(t)
    got = check_all({"q": q, "k": k, "v": v, "dout": dout.transpose(1, 2).contiguous().transpose(1, 2)}, {})
    want = check_all(dict(zip("qkv", dense), dout=dout), {})
    for n in got:
        assert torch.equal(got[n], want[n]), n
    # one key / value sequence for the whole batch
    k1, v1 = (u[:1].expand(2, 4, 90, 16) for u in dense[1:])
    a, _ = attention_forward(dense[0], k1, v1)
    b, _ = attention_forward(dense[0], k1.contiguous(), v1.contiguous())
    assert torch.equal(a, b)
    # an address that 16-byte loads cannot take, and a transposed last axis
    buf = torch.randn(2 * 4 * 90 * 16 + 1, device=device, generator=g).to(t)
    odd = buf[1:].view(2, 4, 90, 16)
    assert torch.equal(attention_forward(odd, dense[1], dense[2])[0], attention_forward(odd.clone(), dense[1], dense[2])[0])
    swap = dense[0].transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(attention_forward(swap, dense[1], dense[2])[0], attention_forward(dense[0], dense[1], dense[2])[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("poison", [math.nan, math.inf])
def test_masked_places_hold_anything(device, dtype, poison):
    """What is masked contributes nothing, also where it shares a tile with what is not."""
    t, kw = inputs(2, 2, 1, 100, 100, 16, TYPES[dtype], 11, bias="coords")
    ids = torch.arange(100, device=device).div(30, rounding_mode="floor").to(torch.int32).repeat(2, 1)
    ids[:, 95:] = -1
    kw["doc_q"] = kw["doc_k"] = ids
    clean = check_all(t, kw, cap=5.0)
    bad = {n: x.clone() for n, x in t.items()}
    for n in bad:
        bad[n][:, :, 95:] = poison                      # padding
    kw["pos_q"][:, 95:] = poison
    got = check_all(bad, kw, cap=5.0)
    for n in got:
        live = slice(None) if n == "dslope" else (slice(None), slice(None), slice(0, 95))
        assert torch.equal(got[n][live], clean[n][live]) or n == "dslope", n
    # another document's values: documents 0, 2, 3 are as before
    other = {n: x.clone() for n, x in t.items()}
    for n in other:
        other[n][:, :, 30:60] = poison
    from dgl_amd.attention import attention_backward, attention_forward
    a = dict(kw, cap=5.0)
    out, lse = attention_forward(other["q"], other["k"], other["v"], **a)
    grads = attention_backward(other["dout"], other["q"], other["k"], other["v"], out, lse, **a)
    # (infinite operands: every capped score is the cap, so the softmax is finite and the infinite values come through)
    assert not out[:, :, 30:60].isfinite().any()
    want = reference(*(torch.where(torch.isfinite(other[n]), other[n], torch.zeros_like(other[n])) for n in ("q", "k", "v", "dout")), **a)
    keep = [i for i in range(95) if not 30 <= i < 60]
    for n, x in (("out", out), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        assert_within(x[:, :, keep], (want[n][0][:, :, keep], want[n][1][:, :, keep]), n)


@pytest.mark.parametrize("dtype", TYPES)
def test_causal_future_holds_anything(device, dtype):
    from dgl_amd.attention import attention_forward
    t, kw = inputs(1, 2, 2, 90, 90, 64, TYPES[dtype], 12)
    clean, _ = attention_forward(t["q"], t["k"], t["v"], causal=True)
    t["v"][:, :, 50:] = math.nan
    t["k"][:, :, 70:] = math.inf
    out, _ = attention_forward(t["q"], t["k"], t["v"], causal=True)
    want = reference(t["q"][:, :, :50], t["k"][:, :, :50], t["v"][:, :, :50], causal=True)
    assert_within(out[:, :, :50], want["out"], "rows before the first NaN")
    assert out[:, :, 50:].isnan().all()
    assert_within(clean[:, :, :50], want["out"], "clean")


def test_empty_shapes(device):
    from dgl_amd.attention import attention, attention_backward, attention_forward
    for B, L, M in ((2, 0, 5), (2, 5, 0), (0, 5, 5), (2, 0, 0)):
        t, kw = inputs(B, 2, 1, L, M, 16, torch.float32, 1, bias="index")
        out, lse = attention_forward(t["q"], t["k"], t["v"], **kw)
        assert out.shape == t["q"].shape and not out.any() and torch.isneginf(lse).all()
        dq, dk, dv, ds = attention_backward(t["dout"], t["q"], t["k"], t["v"], out, lse, **kw)
        assert not dq.any() and not dk.any() and not dv.any() and not ds.any()
        assert dk.shape == t["k"].shape


def test_autograd_matches_the_pair_of_calls_and_differences(device):
    from dgl_amd.attention import attention, attention_backward, attention_forward
    t, kw = inputs(2, 4, 2, 40, 56, 16, torch.float32, 21, bias="coords")
    a = dict(kw, cap=4.0)
    leaves = [t[n].clone().requires_grad_(True) for n in "qkv"] + [kw["slope"].clone().requires_grad_(True)]
    b = dict(a, slope=leaves[3])
    out = attention(*leaves[:3], **b)
    grads = torch.autograd.grad(out, leaves, t["dout"])
    o2, lse = attention_forward(t["q"], t["k"], t["v"], **a)
    pair = attention_backward(t["dout"], t["q"], t["k"], t["v"], o2, lse, **a)
    assert torch.equal(out.detach(), o2)
    for x, y in zip(grads, pair):
        assert torch.equal(x, y)
    # differences of the 64-bit operator along a random direction: the gradient is the formula's and the operator's
    g = torch.Generator(device=device).manual_seed(2)
    along = [torch.randn(x.shape, device=device, generator=g).double() for x in leaves]
    eps = 1e-5
    ends = []
    for sign in (1.0, -1.0):
        x = [u.detach().double() + sign * eps * d for u, d in zip(leaves, along)]
        c = dict(a, slope=x[3])
        s = _value64(x[0], x[1], x[2], **c)
        ends.append((s * t["dout"].double()).sum())
    numeric = float((ends[0] - ends[1]) / (2 * eps))
    analytic = float(sum((x.double() * d).sum() for x, d in zip(grads, along)))
    size = float(sum((x.double() * d).abs().sum() for x, d in zip(grads, along)))
    # binary32 gradients: their bounds are below 1e-4 of the terms' absolute sum; the difference's own error is eps^2
    assert abs(numeric - analytic) <= 1e-5 * size


def _value64(q, k, v, scale=None, cap=0.0, slope=None, pos_q=None, pos_k=None):
    G = q.shape[1] // k.shape[1]
    x = q.shape[-1] ** -0.5 * (q @ k.repeat_interleave(G, 1).transpose(2, 3))
    s = cap * torch.tanh(x / cap) - slope.view(1, -1, 1, 1) * (pos_q.double()[:, :, None] - pos_k.double()[:, None]).norm(dim=-1)[:, None]
    return torch.softmax(s, -1) @ v.repeat_interleave(G, 1)


def test_partial_gradients_and_shared_inputs(device):
    from dgl_amd.attention import attention
    x = torch.randn(1, 2, 50, 16, device=device, requires_grad=True)
    attention(x, x, x).square().sum().backward()               # one tensor three times
    y = x.detach().clone().requires_grad_(True)
    w = torch.softmax(y @ y.transpose(2, 3) / 4, -1) @ y
    w.square().sum().backward()
    torch.testing.assert_close(x.grad, y.grad, rtol=1e-4, atol=1e-4)
    k = torch.randn(1, 1, 50, 16, device=device, requires_grad=True)
    out = attention(x.detach(), k.expand(1, 2, 50, 16), x.detach())   # a broadcast input's gradient is summed by autograd
    out.sum().backward()
    assert k.grad.shape == k.shape and torch.isfinite(k.grad).all()


def test_same_bits_every_time_on_another_stream(device):
    t, kw = inputs(4, 4, 2, 333, 333, 16, torch.float32, 31, bias="coords")
    from dgl_amd.attention import attention_backward, attention_forward
    a = dict(kw, cap=10.0)
    out, lse = attention_forward(t["q"], t["k"], t["v"], **a)
    ref = attention_backward(t["dout"], t["q"], t["k"], t["v"], out, lse, **a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o2, l2 = attention_forward(t["q"], t["k"], t["v"], **a)
        got = attention_backward(t["dout"], t["q"], t["k"], t["v"], o2, l2, **a)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, o2) and all(torch.equal(x, y) for x, y in zip(ref, got))


def test_captured_forward_and_backward_replay(device):
    from dgl_amd.attention import attention, attention_backward, attention_forward
    t, kw = inputs(2, 4, 4, 130, 130, 16, torch.float32, 41, bias="coords")
    a = dict(kw, cap=10.0)

    def both():
        out, lse = attention_forward(t["q"], t["k"], t["v"], **a)
        return (out,) + attention_backward(t["dout"], t["q"], t["k"], t["v"], out, lse, **a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both()
    for seed in (1, 2, 3):
        t["q"].copy_(torch.randn(t["q"].shape, device=device, generator=torch.Generator(device=device).manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        eager = both()
        for x, y in zip(captured, eager):
            assert torch.equal(x, y)
    # a leaf inside a capture is refused (nothing was launched: the capture ends empty)
    leaf = torch.randn(1, 1, 8, 16, device=device, requires_grad=True)
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        with pytest.raises(RuntimeError, match="leaf"):
            attention(leaf, leaf, leaf)
        leaf.detach() * 1.0


def test_gradients_keep_their_types(device):
    from dgl_amd.attention import attention
    slope = torch.full((2,), 0.5, device=device, dtype=torch.bfloat16, requires_grad=True)
    q = torch.randn(1, 2, 20, 16, device=device).bfloat16().requires_grad_(True)
    out = attention(q, q, q, slope=slope)
    out.sum().backward()
    assert q.grad.dtype == torch.bfloat16 and slope.grad.dtype == torch.bfloat16


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,K,L,M,D", [(2, 2, 70, 70, 24), (2, 1, 5, 3000, 16), (4, 1, 300, 130, 128), (16, 16, 2100, 65, 64)])
def test_autograd_in_16_bits(device, dtype, H, K, L, M, D):
    """The differentiable call keeps what the output's rounding left off for its backward pass: one block of rows per wave
    and two, ranges of keys that are joined, head sizes behind the padding."""
    from dgl_amd.attention import attention
    t, kw = inputs(2, H, K, L, M, D, TYPES[dtype], 31, bias="index")
    leaves = [t[n].clone().requires_grad_() for n in "qkv"]
    out = attention(*leaves, **kw)
    out.backward(t["dout"])
    want = reference(t["q"], t["k"], t["v"], t["dout"], **kw)
    assert_within(out.detach(), want["out"], "out")
    for x, n in zip(leaves, ("dq", "dk", "dv")):
        assert_within(x.grad, want[n], n)


def test_rounding_of_the_output_does_not_reach_the_gradients(device):
    """A steep slope: few keys carry a row, and with the output's rounding delta is off by 2^-9 of its terms, as much as the
    score gradients' own rounding (both: sqrt(2) times the error of one); the rest of the output takes that away."""
    from dgl_amd.attention import attention, attention_backward, attention_forward
    t, kw = inputs(2, 4, 4, 512, 512, 64, torch.bfloat16, 37)
    kw["slope"] = torch.full((4,), 0.7, device=device)
    want = reference(t["q"], t["k"], t["v"], t["dout"], **kw)
    leaves = [t[n].clone().requires_grad_() for n in "qkv"]
    attention(*leaves, **kw).backward(t["dout"])
    out, lse = attention_forward(t["q"], t["k"], t["v"], **kw)
    by_hand = attention_backward(t["dout"], t["q"], t["k"], t["v"], out, lse, **kw)
    for n, x, y in zip(("dq", "dk"), leaves, by_hand):
        value = want[n][0]
        error = [((z.double() - value).norm() / value.norm()).item() for z in (x.grad, y)]
        assert error[0] < 0.9 * error[1], (n, error)


def test_wide_ids_and_prefixes_keep_their_sign(device):
    from dgl_amd.attention import attention
    t, _ = inputs(1, 2, 2, 40, 40, 16, torch.float32, 43)
    ids = torch.zeros(1, 40, dtype=torch.int64, device=device)
    ids[:, 30:] = -2 ** 40
    out = attention(t["q"], t["k"], t["v"], doc_q=ids, doc_k=ids)
    assert torch.equal(out, attention(t["q"], t["k"], t["v"], doc_q=ids.clamp(-1).int(), doc_k=ids.clamp(-1).int()))
    assert not out[:, :, 30:].any() and bool(out[:, :, :30].any())
    far = torch.tensor([2 ** 40], device=device)
    assert torch.equal(attention(t["q"], t["k"], t["v"], causal=True, prefix=far),
                       attention(t["q"], t["k"], t["v"], causal=True, prefix=far.clamp(max=40).int()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L,kind", [(1, "one"), (1, "causal"), (5, "documents"), (200, "documents"), (130, "pairs")])
def test_a_single_key_leaves_no_score_gradient(device, dtype, L, kind):
    """A row with one key has the probability 1 whatever its score: dq, dk and dslope are exactly zero where all rows are such,
    dv is dout; beside rows with more keys only they get a gradient."""
    from dgl_amd.attention import attention
    for D, H, K in ((16, 4, 2), (64, 2, 2), (128, 2, 1)):
        t, kw = inputs(2, H, K, L, L, D, TYPES[dtype], L, bias="coords")
        causal = kind == "causal"
        if kind in ("documents", "pairs"):
            ids = torch.arange(L, device=device, dtype=torch.int32).expand(2, L).contiguous()
            if kind == "pairs":
                ids[:, 100:] //= 2
            kw["doc_q"] = kw["doc_k"] = ids
        leaves = [t[n].clone().requires_grad_() for n in "qkv"] + [kw["slope"].clone().requires_grad_()]
        attention(*leaves[:3], **dict(kw, slope=leaves[3], causal=causal, cap=5.0)).backward(t["dout"])
        ids = kw.get("doc_q", torch.zeros(2, L, device=device))[0]
        single = (ids[:, None] == ids[None]).sum(1) == 1           # (halved ids meet some of the first hundred)
        assert not leaves[0].grad[:, :, single].any() and not leaves[1].grad[:, :, single].any()
        assert int(single.sum()) == (85 if kind == "pairs" else L)
        if kind == "pairs":
            assert bool(leaves[0].grad[:, :, ~single].any()) and bool(leaves[1].grad[:, :, ~single].any())
        else:
            assert not leaves[3].grad.any()
        want = reference(t["q"], t["k"], t["v"], t["dout"], cap=5.0, causal=causal, **kw)
        for x, n in zip(leaves, ("dq", "dk", "dv")):
            assert_within(x.grad, want[n], n)
