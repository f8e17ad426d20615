"""Logits processing against the definition: values rounded as the header says, the log-softmax in 64 bits, exact picks."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def values(logits, blocked=None, period=None, bias=None, temperature=1.0, history=None, history_len=None, repetition=1.0,
           presence=0.0, frequency=0.0):
    """The processed values: binary32, one rounding per operation (elementwise torch operations round the same way)."""
    x = logits.float()
    R, A = x.shape
    dev = x.device
    col = lambda t: t.view(-1, 1) if isinstance(t, torch.Tensor) else torch.full((1, 1), t, device=dev)  # noqa: E731
    if history is not None:
        n = history.shape[1]
        live = torch.ones(R, n, dtype=torch.bool, device=dev) if history_len is None else torch.arange(n, device=dev)[None] < history_len[:, None]
        live = live & (history >= 0) & (history < A)
        count = torch.zeros(R, A, device=dev).scatter_add_(1, history.long().clamp(0, A - 1), live.float())
        y = torch.where(x > 0, x / col(repetition), x * col(repetition)) - col(presence)
        x = torch.where(count > 0, y - col(frequency) * count, x)
    if bias is not None:
        x = x + bias
    if temperature != 1.0:
        x = x / torch.full((1, 1), temperature, device=dev)
    if blocked is not None:
        period = period or A
        bits = (((blocked[:, :, None] >> torch.arange(64, device=dev)) & 1) != 0).view(R, -1)
        bits = torch.nn.functional.pad(bits, (0, max(0, period - bits.shape[1])))[:, :period]
        x = torch.where(bits.repeat(1, A // period), -math.inf, x)
    return x


def check(logits, **kw):
    from dgl_amd.logits import process_logits
    log_probs, selected = process_logits(logits, **kw)
    x = values(logits, **kw)
    m = x.amax(1, keepdim=True)
    some = m > -math.inf
    lse = torch.where(some, torch.logsumexp(x.double(), 1, keepdim=True), 0.0)
    want = torch.where(x == -math.inf, -math.inf, x.double() - lse)
    dead = torch.isinf(want)
    assert torch.equal(torch.isinf(log_probs), dead)
    # exponentials: their argument is rounded three times (d e^-d < 0.4), sums: 32 terms a thread, 10 levels above, up to
    # 128 tiles; logarithm and the two subtractions round values of the size of x, its maximum and lse
    top = torch.where(some, m.double().abs(), 0.0)
    bound = U * (3 + 2 + 32 + 10 + 128) + 3 * U * (torch.where(dead, 0.0, x.double()).abs() + lse.abs() + top)
    off = torch.where(dead, 0.0, (log_probs.double() - want).abs())
    assert bool((off <= bound).all()), f"off by {float((off / bound).max()):.3g} bounds"
    first = torch.where(x == m, torch.arange(x.shape[1], device=x.device), x.shape[1]).amin(1)
    assert torch.equal(selected, torch.where(some[:, 0], first, -1).to(torch.int32))
    return log_probs, selected


def rnd(R, A, dtype, seed, device="cuda", scale=3.0):
    g = torch.Generator(device=device).manual_seed(seed)
    return (scale * torch.randn(R, A, device=device, generator=g)).to(dtype), g


def words(R, n, g, device="cuda"):
    return torch.randint(-2 ** 62, 2 ** 62, (R, (n + 63) // 64), device=device, generator=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("A", [1, 2, 63, 64, 255, 256, 257, 1000, 1023, 4096, 4097, 8192, 8193, 16384, 16390, 32768, 32769, 40000, 70001])
def test_sizes(device, dtype, A):
    x, g = rnd(3, A, TYPES[dtype], A)
    check(x)
    hist = torch.randint(0, A, (3, 50), device=device, generator=g).to(torch.int32)
    check(x, blocked=words(3, A, g), bias=torch.randn(A, device=device, generator=g), temperature=0.7, history=hist,
          history_len=torch.tensor([50, 0, 13], device=device, dtype=torch.int32),
          repetition=torch.tensor([1.3, 1.1, 0.8], device=device), presence=torch.rand(3, device=device, generator=g),
          frequency=torch.rand(3, device=device, generator=g))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("A,period", [(202, 101), (20002, 10001), (66, 1), (40002, 6667), (40004, 2)])
def test_actions_that_share_bits(device, dtype, A, period):
    x, g = rnd(5, A, TYPES[dtype], A)
    blocked = words(5, period, g)
    blocked[0] = -1
    lp, sel = check(x, blocked=blocked, period=period)
    assert sel[0] == -1 and torch.isneginf(lp[0]).all()


@pytest.mark.parametrize("A", [100, 5000, 50000])
def test_penalties(device, A):
    x, g = rnd(4, A, torch.float32, 1)
    hist = torch.randint(-3, A + 3, (4, 300), device=device, generator=g).to(torch.int32)      # entries outside are ignored
    hist[1] = 5                                                                                # one action 300 times
    check(x, history=hist, repetition=1.2, presence=0.5, frequency=0.01)
    check(x, history=hist, repetition=0.5)
    check(x, history=hist, history_len=torch.tensor([-1, 300, 1000, 7], device=device, dtype=torch.int32), frequency=2.0)
    check(x, history=hist[:, :0])


@pytest.mark.parametrize("temperature", [0.7, 1.0 / 3.0, 1.9999998807907104, 1e-3, 37.5, 1e35])
def test_temperature_divides_exactly(device, temperature):
    """Equal quotients tie, so a pick depends on the division's last bit: 200 000 values in 100 rows of near-ties."""
    g = torch.Generator(device=device).manual_seed(6)
    x = 1.0 + torch.randint(0, 8, (100, 2000), device=device, generator=g) * 2.0 ** -23
    x = x * torch.exp2(torch.randint(-60, 60, (100, 1), device=device, generator=g).float())
    check(x, temperature=temperature)


def test_many_repeats_count_in_full(device):
    """Histories of 65536 entries and more count in 32 bits."""
    x, g = rnd(2, 300, torch.float32, 8)
    for n in (65535, 65536, 70000):
        check(x, history=torch.full((2, n), 17, device=device, dtype=torch.int32), frequency=1e-4)


def test_equal_logits_go_to_the_lowest_action(device):
    for A in (7, 1000, 5000, 50000):
        x = torch.zeros(3, A, device=device)
        x[1, A // 2:] = 1.0
        x[2, -1] = 1.0
        _, sel = check(x)
        assert sel.tolist() == [0, A // 2, A - 1]


@pytest.mark.parametrize("A", [50, 3000, 40000])
def test_special_values(device, A):
    from dgl_amd.logits import process_logits
    x, g = rnd(5, A, torch.float32, 2)
    x[0] = torch.finfo(torch.float32).min                # a mask written as the type's lowest value: a flat row
    x[1, : A // 2] = -math.inf
    x[2, 3] = 3e38
    x[3] = 1e30
    check(x)
    blocked = torch.zeros(5, (A + 63) // 64, dtype=torch.int64, device=device)
    blocked[:, 0] = 1 << 4
    y = x.clone()
    y[:, 4] = math.nan                                   # blocked places hold anything
    lp, sel = process_logits(y, blocked=blocked)
    ref, ref_sel = process_logits(x, blocked=blocked)
    assert torch.equal(lp, ref) and torch.equal(sel, ref_sel)
    y[4, 7] = math.nan                                   # a live NaN makes its row NaN, and is never picked
    lp, sel = process_logits(y, blocked=blocked)
    assert lp[4, 0].isnan() and torch.equal(lp[:4], ref[:4]) and sel[4] == ref_sel[4]


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(device, dtype):
    from dgl_amd.logits import process_logits
    x, g = rnd(6, 2 * 1001, TYPES[dtype], 3)
    assert torch.equal(process_logits(x[:, 1:1002])[0], process_logits(x[:, 1:1002].contiguous())[0])
    assert torch.equal(process_logits(x[::2, ::2])[0], process_logits(x[::2, ::2].contiguous())[0])
    one = x[:1].expand(4, -1)
    assert torch.equal(process_logits(one)[0], process_logits(one.contiguous())[0])
    b = torch.randn(6, 2 * 1001, device=device, generator=g)
    # (rows that 16-byte accesses cannot take are read value by value: their sums run in another order, so the definition
    # and not the copy's bits is what they are held to)
    check(x[:, :1000], bias=b[:, 3:1003])
    check(x[:, 1:1001], bias=b[:, 3:1003])


def test_captured_calls_replay(device):
    from dgl_amd.logits import process_logits
    for A in (1000, 50000):
        x, g = rnd(8, A, torch.float32, 4)
        hist = torch.randint(0, A, (8, 64), device=device, generator=g).to(torch.int32)
        live = torch.full((8,), 10, device=device, dtype=torch.int32)
        blocked = words(8, A, g)
        call = lambda: process_logits(x, blocked=blocked, history=hist, history_len=live, frequency=0.5)  # noqa: E731
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lp, sel = call()
        for _ in range(3):
            x.mul_(0.9)
            live.add_(9)
            blocked.bitwise_xor_(1 << 9)
            graph.replay()
            torch.cuda.synchronize()
            a, b = call()
            assert torch.equal(lp, a) and torch.equal(sel, b)


def test_refusals(device):
    from dgl_amd._lib import DglError
    from dgl_amd.logits import process_logits
    x = torch.zeros(2, 10, device=device)
    for kw in ({"blocked": torch.zeros(2, 1, device=device)}, {"blocked": torch.zeros(3, 1, device=device, dtype=torch.int64)},
               {"bias": torch.zeros(9, device=device)}, {"history_len": torch.zeros(2, device=device, dtype=torch.int32)},
               {"history": torch.zeros(10, device=device, dtype=torch.int32)}, {"repetition": torch.ones(3, device=device)}):
        with pytest.raises(ValueError):
            process_logits(x, **kw)
    for kw in ({"temperature": 0.0}, {"temperature": math.nan}, {"blocked": torch.zeros(2, 1, device=device, dtype=torch.int64), "period": 3},
               {"history": torch.zeros(2, 3, device=device, dtype=torch.int32), "repetition": 0.0}):
        with pytest.raises(DglError):
            process_logits(x, **kw)
    with pytest.raises(ValueError):
        process_logits(x.cpu())
    assert process_logits(x[:0])[0].shape == (0, 10)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("A,period", [(70, 7), (33, 33), (96, 3), (4095, 45), (24570, 819), (24576, 24576), (40000, 10000), (49149, 16383)])
def test_bits_of_any_period(device, dtype, A, period):
    """Periods that end inside a word, in the middle of a tile, and several times within 32 actions; bits beyond the words
    that are given are clear; with a history beside them."""
    x, g = rnd(4, A, TYPES[dtype], A + period)
    blocked = words(4, period, g)
    check(x, blocked=blocked, period=period)
    hist = torch.randint(0, A, (4, 70), device=device, generator=g).to(torch.int32)
    check(x, blocked=blocked[:, : max(1, blocked.shape[1] // 2)], period=period, history=hist, presence=0.5, frequency=0.25)


def test_wide_history_entries_are_no_actions(device):
    from dgl_amd.logits import process_logits
    x, g = rnd(2, 100, torch.float32, 3)
    history = torch.tensor([[5, 7, 2 ** 32 + 5, -2 ** 33 + 9], [2 ** 31, 2 ** 40, -1, 3]], device=device)
    narrow = torch.tensor([[5, 7, -1, -1], [-1, -1, -1, 3]], device=device, dtype=torch.int32)
    for a, b in zip(process_logits(x, history=history, presence=1.0), process_logits(x, history=narrow, presence=1.0)):
        assert torch.equal(a, b)
