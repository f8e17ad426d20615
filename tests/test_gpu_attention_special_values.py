"""NaN and infinities in places that are seen, with scores capped on both sides of the precise tanh's threshold (64): they
come out as the definition has them, from the attention operator, its gradients and the single-token form."""
import math

import pytest
import torch

from attention_reference import U, assert_within, half_step, reference

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CAPS = [0.5, 10.0, 64.0, 65.0, 1000.0]


def qkv(B, H, K, L, M, D, dtype, seed, device):
    g = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=device, generator=g).to(dtype)  # noqa: E731
    return rnd(B, H, L, D), rnd(B, K, M, D), rnd(B, K, M, D), rnd(B, H, L, D)


def saturated(scores, v, err, dtype):
    """softmax(scores) v with the bound of the operator for scores that are off by `err`: it enters a probability twice (own
    score, row sum), the sums of M terms add U (64 + M), 16-bit types round p (half precision: at least by 2^-25 of the row's
    largest) and everything rounds the output."""
    M = scores.shape[-1]
    p = torch.softmax(scores, -1)
    h = 0.0 if dtype == torch.float32 else half_step(dtype)
    out = p @ v
    bound = (p * (2 * err + U * (64 + M) + h)) @ v.abs() + half_step(dtype) * out.abs() * 1.01 + 1e-30
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25 * (p.amax(-1, keepdim=True) * torch.ones_like(p)) @ v.abs() + 2.0 ** -25
    return out, bound


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0] + CAPS)
@pytest.mark.parametrize("D,M", [(16, 70), (64, 70), (128, 200), (16, 3000)])
def test_a_nan_query_row_is_nan(device, dtype, cap, D, M):
    """The row of the NaN query alone: output, lse and dq; through it dk and dv of every key it sees."""
    from dgl_amd.attention import attention_backward, attention_forward
    q, k, v, do = qkv(1, 2, 1, 70, M, D, TYPES[dtype], 1, device)
    q[0, 1, 33, 5] = math.nan
    out, lse = attention_forward(q, k, v, cap=cap)
    assert out[0, 1, 33].isnan().all() and lse[0, 1, 33].isnan()
    keep = [i for i in range(70) if i != 33]
    want = reference(q.nan_to_num(0.0), k, v, cap=cap)
    assert_within(out[:, :, keep], tuple(x[:, :, keep] for x in want["out"]), "out")
    assert_within(lse[:, :, keep], tuple(x[:, :, keep] for x in want["lse"]), "lse")
    dq, dk, dv, _ = attention_backward(do, q, k, v, out, lse, cap=cap)
    assert dq[0, 1, 33].isnan().all() and dq[:, :, keep].isfinite().all()
    assert dk.isnan().all() and dv.isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0] + CAPS)
@pytest.mark.parametrize("D", [16, 64, 128])
def test_a_nan_key_reaches_the_rows_that_see_it(device, dtype, cap, D):
    from dgl_amd.attention import attention_backward, attention_forward
    q, k, v, do = qkv(1, 2, 2, 150, 150, D, TYPES[dtype], 2, device)
    k[0, 0, 77, 3] = math.nan
    out, lse = attention_forward(q, k, v, cap=cap, causal=True)
    assert out[0, 0, 77:].isnan().all() and lse[0, 0, 77:].isnan().all()
    want = reference(q, k.nan_to_num(0.0), v, cap=cap, causal=True)
    assert_within(out[0, 0, :77], tuple(x[0, 0, :77] for x in want["out"]), "rows before the key")
    assert_within(out[0, 1], tuple(x[0, 1] for x in want["out"]), "the other head")
    dq, dk, dv, _ = attention_backward(do, q, k, v, out, lse, cap=cap, causal=True)
    assert dq[0, 0, 77:].isnan().all() and dq[0, 0, :77].isfinite().all() and dq[0, 1].isfinite().all()
    assert dk[0, 0].isnan().all() and dv[0, 0].isnan().all() and dk[0, 1].isfinite().all() and dv[0, 1].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", CAPS[1:])
@pytest.mark.parametrize("D,M", [(16, 70), (128, 200), (16, 3000)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_infinite_operands_saturate_the_cap(device, dtype, cap, D, M, sign):
    """One infinite element of a query: its scores are the cap with the sign of the key's element.  One of a key: the score
    of every row against it is the cap with the sign of the row's element."""
    from dgl_amd.attention import attention_backward, attention_forward
    q, k, v, do = qkv(1, 1, 1, 66, M, D, TYPES[dtype], 3, device)
    far = q.clone()
    far[0, 0, 40, 2] = sign * math.inf
    out, lse = attention_forward(far, k, v, cap=cap)
    s = cap * sign * torch.sign(k[0, 0, :, 2].double())
    assert s.abs().min() == cap
    err = 32 * U * cap                              # the cap itself in units of log2, and its tanh
    assert_within(out[0, 0, 40:41], saturated(s[None], v[0, 0].double(), err, TYPES[dtype]), "the infinite query's row")
    assert abs(float(lse[0, 0, 40]) - float(torch.logsumexp(s, 0))) <= err + U * (64 + M) + 4 * U * cap
    dq = attention_backward(do, far, k, v, out, lse, cap=cap)[0]
    assert not dq[0, 0, 40].any()                   # a saturated tanh has no slope
    far = k.clone()
    far[0, 0, 7, 2] = sign * math.inf
    out, lse = attention_forward(q, far, v, cap=cap)
    x = D ** -0.5 * (q[0, 0].double() @ k[0, 0].double().T)
    size = D ** -0.5 * (q[0, 0].double().abs() @ k[0, 0].double().abs().T)
    s = cap * torch.tanh(x / cap)
    s[:, 7] = cap * sign * torch.sign(q[0, 0, :, 2].double())
    err = (U * ((D + 8) * size + 32 * cap)).amax(-1, keepdim=True)
    assert_within(out[0, 0], saturated(s, v[0, 0].double(), err, TYPES[dtype]), "rows that see an infinite key")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [0.0] + CAPS)
@pytest.mark.parametrize("n,D", [(90, 16), (90, 128), (5000, 16)])
def test_single_token_form(device, dtype, cap, n, D):
    """A NaN query head; a NaN in a key that two of three rows see; an infinite element of a query."""
    from dgl_amd.attention import PagedCache, attention_step
    t = TYPES[dtype]
    g = torch.Generator(device=device).manual_seed(4)
    k, v = (torch.randn(1, 1, n, D, device=device, generator=g).to(t) for _ in range(2))
    q = torch.randn(3, 2, D, device=device, generator=g).to(t)
    cache = PagedCache(1, 1, D, n, page_size=32, dtype=t, device=device)
    cache.append(k, v)
    bad = q.clone()
    bad[1, 1, 4] = math.nan
    out, lse = attention_step(bad, cache, rows_per_instance=3, cap=cap, return_lse=True)
    want = reference(q.transpose(0, 1)[None], k, v, cap=cap)
    clean = torch.ones(3, 2, dtype=torch.bool, device=device)
    clean[1, 1] = False
    assert out[1, 1].isnan().all() and lse[1, 1].isnan()
    for got, name in ((out, "out"), (lse, "lse")):
        assert_within(got[clean], tuple(x[0].transpose(0, 1)[clean] for x in want[name]), name)
    if cap > 1.0:
        far = q.clone()
        far[2, 0, 1] = -math.inf
        got = attention_step(far, cache, rows_per_instance=3, cap=cap)
        s = -cap * torch.sign(k[0, 0, :, 1].double())
        assert s.abs().min() == cap
        assert_within(got[2, 0][None], saturated(s[None], v[0, 0].double(), 32 * U * cap, t), "an infinite query")
    k[0, 0, 9, 0] = math.nan
    cache = PagedCache(1, 1, D, n, page_size=32, dtype=t, device=device)
    cache.append(k, v)
    blocked = torch.zeros(3, (n + 63) // 64, dtype=torch.int64, device=device)
    blocked[0, 0] = 1 << 9
    out, lse = attention_step(q, cache, rows_per_instance=3, cap=cap, blocked=blocked, return_lse=True)
    assert out[1:].isnan().all() and lse[1:].isnan().all() and out[0].isfinite().all() and lse[0].isfinite().all()
