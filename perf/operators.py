"""Attention over nodes and sequences, attention of single tokens over a paged cache, and logits processing: cases,
plain forms and exact values.

Three operators, from encoding an instance to choosing its next node:

``attention``  multi-head attention with scores capped by a tanh, a bias that falls with distance (between 2-D node
               coordinates, or between positions of a sequence), document, causal and prefix masks; forward alone
               (an encoder that serves) or forward and backward (a training step).
``step``       one new token per row against the pages of its instance's key-value cache; the rows of an instance
               (multi-starts x beams) share its pages, each row has its own blocked (visited) bits.
``logits``     penalties for repeated actions, biases, temperature and blocked actions on a batch of logits, ending in
               log-probabilities and the greedy pick.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------------------- cases
def _attention(name, dtype, batch, heads, kv_heads, length, dim, *, keys=0, cap=0.0, bias="none", docs=0, causal=False,
               prefix=0, train=False):
    return {"name": name, "op": "attention", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "length": length, "keys": keys or length, "dim": dim, "cap": cap, "bias": bias, "docs": docs,
            "causal": causal, "prefix": prefix, "train": train}


def _step(name, dtype, batch, rows, heads, kv_heads, length, dim, *, page=64, cap=0.0, bias="none", blocked=True,
          ragged=False, append=False):
    return {"name": name, "op": "step", "dtype": dtype, "batch": batch, "rows": rows, "heads": heads,
            "kv_heads": kv_heads, "length": length, "dim": dim, "page": page, "cap": cap, "bias": bias,
            "blocked": blocked, "ragged": ragged, "append": append}


def _logits(name, dtype, rows, actions, *, blocked=True, period=0, history=0, bias="none", temperature=1.0,
            penalties=False):
    return {"name": name, "op": "logits", "dtype": dtype, "rows": rows, "actions": actions, "blocked": blocked,
            "period": period or actions, "history": history, "bias": bias, "temperature": temperature,
            "penalties": penalties}


def listed():
    return [
        # an encoder layer over a small batch of 100-node instances with the policy's heads (8 of 16): latency
        _attention("nodes_100", "f32", 16, 8, 8, 100, 16, cap=10.0, bias="coords"),
        # the same over 1000-node instances: the headline size of the decode benchmark
        _attention("nodes_1000", "f32", 64, 8, 8, 1000, 16, cap=10.0, bias="coords"),
        # a training step on CVRP-1000 (depot + customers) whose rows hold several instances packed one after another
        _attention("train_packed_1001", "f32", 8, 8, 8, 1001, 16, cap=10.0, bias="coords", docs=4, train=True),
        # a training step of a sequence decoder with a prefix it reads in full, distance bias and shared key heads
        _attention("train_prefix_2047", "bf16", 2, 16, 4, 2047, 64, bias="index", causal=True, prefix=500, train=True),
        # packed documents of ragged sizes, half precision, no cap, no bias
        _attention("train_docs_6000", "f16", 1, 8, 8, 6000, 64, docs=9, train=True),
        # a long prompt, causal, capped scores, wide heads
        _attention("prompt_8192", "bf16", 1, 32, 8, 8192, 128, cap=30.0, causal=True),
        # one decoding step of a single 100-node instance: the smallest call of a serving loop
        _step("step_100", "f32", 1, 1, 8, 8, 100, 16, cap=10.0, bias="coords"),
        # one step of beam search (16 beams) over a batch of 1000-node instances
        _step("step_1000_beam16", "f32", 32, 16, 8, 8, 1000, 16, cap=10.0, bias="coords"),
        # one step of a token generator over long ragged caches; the new token's keys and values are appended first
        _step("step_65536", "bf16", 8, 1, 32, 8, 65536, 128, cap=30.0, blocked=False, ragged=True, append=True),
        # one decision of a greedy rollout of 512 TSP-1000 instances: visited nodes blocked
        _logits("logits_1000", "f32", 512, 1000),
        # CVRP-10000: direct and via-depot actions share the visited bits, node biases, penalties on chosen nodes
        _logits("logits_20002", "f32", 512, 20002, period=10001, history=64, bias="actions", temperature=0.7,
                penalties=True),
        # a large vocabulary in bfloat16 with a long history
        _logits("logits_131072", "bf16", 256, 131072, history=2048, temperature=1.3, penalties=True),
    ]


def _between(rng, lo, hi):
    """Spread over the logarithm of the range, odd numbers as often as even ones."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "step", "step", "logits"])
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    dim = rng.choice([16, 32, 64, 128])
    if op == "logits":
        actions = _between(rng, 2, 131072)
        rows = _between(rng, 1, max(1, min(2048, (256 * 131072) // actions // 2)))
        period = actions // 2 if actions % 2 == 0 and rng.random() < 0.3 else actions
        c = _logits("", dtype, rows, actions, blocked=rng.random() < 0.8, period=period,
                    history=rng.choice([0, _between(rng, 1, 2048)]), bias=rng.choice(["none", "actions", "rows"]),
                    temperature=rng.choice([1.0, 0.6, 1.7]), penalties=rng.random() < 0.6)
    elif op == "step":
        groups = rng.choice([1, 1, 4, 8])
        kv = rng.choice([1, 2, 8])
        length = _between(rng, 1, 65536)
        most = (8 * 65536 * 8 * 128) // (length * kv * dim) // 2
        batch = _between(rng, 1, max(1, min(64, most)))
        rows = _between(rng, 1, max(1, min(100, 4096 // groups, (1 << 28) // (batch * length * kv * groups))))
        c = _step("", dtype, batch, rows, kv * groups, kv, length, dim, page=rng.choice([16, 32, 64, 128]),
                  cap=rng.choice([0.0, 10.0, 30.0]), bias=rng.choice(["none", "index", "coords"]),
                  blocked=rng.random() < 0.6, ragged=rng.random() < 0.5, append=rng.random() < 0.4)
    else:
        train = rng.random() < 0.5
        groups = rng.choice([1, 1, 2, 4])
        kv = rng.choice([1, 2, 8])
        length = _between(rng, 1, 6000)
        keys = length if train or rng.random() < 0.7 else _between(rng, 1, 6000)
        most = (1 << 28) * 16 // (length * keys * kv * groups * dim) // (4 if train else 1)
        batch = _between(rng, 1, max(1, min(128, most)))
        causal = rng.random() < 0.4
        c = _attention("", dtype, batch, kv * groups, kv, length, dim, keys=keys, cap=rng.choice([0.0, 10.0, 30.0]),
                       bias=rng.choice(["none", "index", "coords"]), docs=rng.choice([0, 0, 3, 7]) if keys == length else 0,
                       causal=causal, prefix=rng.choice([0, keys // 3]) if causal else 0, train=train)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _slopes(case):
    """Coordinates lie in the unit square; positions are whole numbers: gentle slopes there."""
    h = torch.arange(case["heads"], device=DEV, dtype=torch.float32)
    return 0.5 * (1.0 + h) if case["bias"] == "coords" else torch.exp2(-8.0 * (h + 1.0) / case["heads"])


def _documents(case, g):
    """Ragged documents one after another, and a few padding tokens (-1) at the end of every row but the first."""
    B, L = case["batch"], case["length"]
    cuts = torch.randint(0, L, (B, case["docs"] - 1), device=DEV, generator=g)
    ids = (torch.arange(L, device=DEV)[None, :, None] >= cuts[:, None, :]).sum(-1)
    pad = torch.arange(B, device=DEV) * 3 % max(1, L // 2)
    return torch.where(torch.arange(L, device=DEV)[None] >= L - pad[:, None], -1, ids).to(torch.int32).contiguous()


def _prepare_attention(case, seed):
    g, t = _gen(seed), TYPES[case["dtype"]]
    B, H, K, L, M, D = (case[n] for n in ("batch", "heads", "kv_heads", "length", "keys", "dim"))
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g).to(t)  # noqa: E731
    # token-major storage, as the linear layers before the operator leave it: heads are a strided axis
    s = {"q": rnd(B, L, H, D).transpose(1, 2), "k": rnd(B, M, K, D).transpose(1, 2), "v": rnd(B, M, K, D).transpose(1, 2)}
    s["scale"], s["cap"], s["causal"] = 1.0 / math.sqrt(D), case["cap"], case["causal"]
    s["slope"] = _slopes(case) if case["bias"] != "none" else None
    s["pos_q"] = s["pos_k"] = s["doc_q"] = s["doc_k"] = s["prefix"] = None
    if case["bias"] == "coords":
        s["pos_k"] = torch.rand(B, M, 2, device=DEV, generator=g)
        s["pos_q"] = s["pos_k"] if L == M else torch.rand(B, L, 2, device=DEV, generator=g)
    if case["docs"]:
        s["doc_q"] = s["doc_k"] = _documents(case, g)
    if case["prefix"]:
        s["prefix"] = torch.randint(0, case["prefix"] + 1, (B,), device=DEV, generator=g).to(torch.int32)
    if case["train"]:
        s["dout"] = rnd(B, L, H, D).transpose(1, 2)
        for n in ("q", "k", "v", "slope"):
            if s[n] is not None:
                s[n].requires_grad_(True)
    return s


def _blocked(rows, n, g):
    """Bits as the state's visited words hold them: bit j of word j // 64; about half are set, one row has all."""
    bits = torch.rand(rows, (n + 63) // 64 * 64, device=DEV, generator=g) < 0.5
    if rows > 4:
        bits[3] = True
    shift = torch.arange(64, device=DEV)
    return (bits.view(rows, -1, 64).to(torch.int64) << shift).sum(-1)


def _prepare_step(case, seed):
    g, t = _gen(seed), TYPES[case["dtype"]]
    B, P, H, K, N, D, page = (case[n] for n in ("batch", "rows", "heads", "kv_heads", "length", "dim", "page"))
    per = (N + page - 1) // page
    s = {"q": torch.randn(B * P, H, D, device=DEV, generator=g).to(t), "rows": P, "page": page}
    total = B * per + 3
    s["k_pages"] = torch.randn(total, K, page, D, device=DEV, generator=g).to(t)
    s["v_pages"] = torch.randn(total, K, page, D, device=DEV, generator=g).to(t)
    s["table"] = torch.randperm(total, device=DEV, generator=g)[:B * per].view(B, per).to(torch.int32)
    low = max(1, N // 2) if case["ragged"] else N
    s["lengths"] = torch.randint(low, N + 1, (B,), device=DEV, generator=g).to(torch.int32)
    s["scale"], s["cap"] = 1.0 / math.sqrt(D), case["cap"]
    s["slope"] = _slopes(case) if case["bias"] != "none" else None
    s["pos_q"] = s["pos_k"] = s["blocked"] = s["k_new"] = s["v_new"] = None
    if case["bias"] == "coords":
        s["pos_k"] = torch.rand(B, N, 2, device=DEV, generator=g)
        s["pos_q"] = torch.rand(B * P, 2, device=DEV, generator=g)
    if case["blocked"]:
        s["blocked"] = _blocked(B * P, N, g)
    if case["append"]:
        # the last live token of every sequence is the one that this pass brings
        s["k_new"] = torch.randn(B, K, 1, D, device=DEV, generator=g).to(t)
        s["v_new"] = torch.randn(B, K, 1, D, device=DEV, generator=g).to(t)
        s["start"] = s["lengths"] - 1
    return s


def _prepare_logits(case, seed):
    g, t = _gen(seed), TYPES[case["dtype"]]
    R, A, L = case["rows"], case["actions"], case["history"]
    s = {"logits": (3.0 * torch.randn(R, A, device=DEV, generator=g)).to(t), "period": case["period"],
         "temperature": case["temperature"], "blocked": None, "bias": None, "history": None, "history_len": None,
         "repetition": None, "presence": None, "frequency": None}
    if case["blocked"]:
        s["blocked"] = _blocked(R, case["period"], g)
    if case["bias"] != "none":
        s["bias"] = torch.randn(*((A,) if case["bias"] == "actions" else (R, A)), device=DEV, generator=g)
    if L:
        # squares crowd the low actions: repeated ones are met
        s["history"] = (torch.rand(R, L, device=DEV, generator=g).square() * A).to(torch.int32).clamp_(max=A - 1)
        s["history_len"] = torch.randint(0, L + 1, (R,), device=DEV, generator=g).to(torch.int32)
    if case["penalties"]:
        s["repetition"] = 1.0 + 0.5 * torch.rand(R, device=DEV, generator=g)
        s["presence"] = torch.rand(R, device=DEV, generator=g)
        s["frequency"] = 0.3 * torch.rand(R, device=DEV, generator=g)
    return s


def prepare(case, seed):
    with torch.no_grad():
        s = {"attention": _prepare_attention, "step": _prepare_step, "logits": _prepare_logits}[case["op"]](case, seed)
    s["op"], s["train"] = case["op"], case.get("train", False)
    return s


# ------------------------------------------------------------------------------------------------------- plain forms
def _distance(pos_q, pos_k):
    d = pos_q[:, :, None, :] - pos_k[:, None, :, :]
    return torch.sqrt(d[..., 0] * d[..., 0] + d[..., 1] * d[..., 1])


def _softmax(s):
    """Rows without a finite score are zero."""
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0)


def _plain_attention(s):
    q, k, v = s["q"].detach().float(), s["k"].detach().float(), s["v"].detach().float()
    (B, H, L, D), K, M = q.shape, k.shape[1], k.shape[2]
    G = H // K
    q = q.reshape(B, K, G * L, D)
    x = torch.matmul(q, k.transpose(2, 3)).view(B, K, G, L, M) * s["scale"]
    th = None
    if s["cap"] > 0:
        th = torch.tanh(x / s["cap"])
        x = s["cap"] * th
    dist = None
    i, j = torch.arange(L, device=DEV)[:, None] + (M - L), torch.arange(M, device=DEV)[None]
    if s["slope"] is not None:
        dist = _distance(s["pos_q"], s["pos_k"])[:, None, None] if s["pos_q"] is not None else (i - j).abs().float()[None, None, None]
        x = x - s["slope"].detach().view(1, K, G, 1, 1) * dist
    keep = None
    if s["causal"]:
        keep = (j <= i)[None] if s["prefix"] is None else (j <= i)[None] | (j[None] < s["prefix"][:, None, None])
    if s["doc_q"] is not None:
        same = (s["doc_q"][:, :, None] == s["doc_k"][:, None, :]) & (s["doc_k"] >= 0)[:, None, :]
        keep = same if keep is None else keep & same
    if keep is not None:
        x = torch.where(keep[:, None, None], x, -math.inf)
    p = _softmax(x)
    del x
    out = torch.matmul(p.view(B, K, G * L, M), v).view(B, H, L, D).to(s["q"].dtype)
    if not s["train"]:
        return {"out": out}
    do = s["dout"].float().reshape(B, K, G * L, D)
    dp = torch.matmul(do, v.transpose(2, 3)).view(B, K, G, L, M)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    got = {"out": out}
    if dist is not None:
        got["dslope"] = -(ds * dist).sum((0, 3, 4), dtype=torch.float64).view(H).float()
    if th is not None:
        ds = ds * (1.0 - th * th)
    ds = (ds * s["scale"]).view(B, K, G * L, M)
    t = s["q"].dtype
    got["dq"] = torch.matmul(ds, k).view(B, H, L, D).to(t)
    got["dk"] = torch.matmul(ds.transpose(2, 3), q).to(t)
    got["dv"] = torch.matmul(p.view(B, K, G * L, M).transpose(2, 3), do).to(t)
    return got


def _plain_step(s):
    q = s["q"].float()
    (R, H, D), P, page = q.shape, s["rows"], s["page"]
    B, per = s["table"].shape
    K = s["k_pages"].shape[1]
    table, lengths = s["table"].long(), s["lengths"].long()
    if s["k_new"] is not None:
        at = s["start"].long()
        pages = table.gather(1, (at // page)[:, None])[:, 0]
        s["k_pages"][pages, :, at % page] = s["k_new"][:, :, 0]
        s["v_pages"][pages, :, at % page] = s["v_new"][:, :, 0]
    n = per * page
    k = s["k_pages"][table].transpose(1, 2).reshape(B, K, n, D).float()
    v = s["v_pages"][table].transpose(1, 2).reshape(B, K, n, D).float()
    G = H // K
    x = torch.matmul(q.view(B, P, K, G, D).transpose(1, 2).reshape(B, K, P * G, D), k.transpose(2, 3))
    x = x.view(B, K, P, G, n) * s["scale"]
    if s["cap"] > 0:
        x = s["cap"] * torch.tanh(x / s["cap"])
    j = torch.arange(n, device=DEV)
    if s["slope"] is not None:
        if s["pos_q"] is not None:
            pos = torch.nn.functional.pad(s["pos_k"], (0, 0, 0, n - s["pos_k"].shape[1]))
            dist = _distance(s["pos_q"].view(B, P, 2), pos)[:, None, :, None]
        else:
            dist = (lengths[:, None] - 1 - j[None]).abs().float()[:, None, None, None]
        x = x - s["slope"].view(1, K, 1, G, 1) * dist
    keep = (j[None] < lengths[:, None])[:, None, None, None]
    if s["blocked"] is not None:
        bits = (s["blocked"][:, :, None] >> torch.arange(64, device=DEV)) & 1
        bits = torch.nn.functional.pad(bits.view(R, -1), (0, max(0, n - 64 * s["blocked"].shape[1])))[:, :n]
        keep = keep & (bits == 0).view(B, 1, P, 1, n)
    p = _softmax(torch.where(keep, x, -math.inf))
    out = torch.matmul(p.view(B, K, P * G, n), v).view(B, K, P, G, D).transpose(1, 2).reshape(R, H, D).to(s["q"].dtype)
    return {"out": out, "k_pages": s["k_pages"], "v_pages": s["v_pages"]} if s["k_new"] is not None else {"out": out}


def _plain_logits(s):
    x = s["logits"].float()
    R, A = x.shape
    if s["history"] is not None and s["repetition"] is not None:
        L = s["history"].shape[1]
        live = (torch.arange(L, device=DEV)[None] < s["history_len"][:, None]).float()
        count = torch.zeros(R, A, device=DEV).scatter_add_(1, s["history"].long(), live)
        rep = s["repetition"][:, None]
        y = torch.where(x > 0, x / rep, x * rep) - s["presence"][:, None]
        x = torch.where(count > 0, y - s["frequency"][:, None] * count, x)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["temperature"] != 1.0:
        # by a tensor: a division, not a product with a rounded reciprocal
        x = x / torch.full((1, 1), s["temperature"], device=DEV)
    if s["blocked"] is not None:
        bits = ((s["blocked"][:, :, None] >> torch.arange(64, device=DEV)) & 1).view(R, -1)[:, :s["period"]]
        x = torch.where(bits.repeat(1, A // s["period"]) == 0, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    lse = torch.where(m == -math.inf, 0.0, m) + torch.log(e.sum(-1, keepdim=True))
    first = torch.where(x == m, torch.arange(A, device=DEV), A).amin(-1)
    selected = torch.where(m[:, 0] == -math.inf, -1, first).to(torch.int32)
    return {"log_probs": torch.where(x == -math.inf, -math.inf, x - lse), "selected": selected}


# --------------------------------------------------------------------------------------------------- the framework's
def _own_attention(s):
    from dgl_amd.attention import attention
    out = attention(s["q"], s["k"], s["v"], scale=s["scale"], cap=s["cap"], slope=s["slope"], pos_q=s["pos_q"],
                    pos_k=s["pos_k"], doc_q=s["doc_q"], doc_k=s["doc_k"], causal=s["causal"], prefix=s["prefix"])
    if not s["train"]:
        return {"out": out}
    wrt = [n for n in ("q", "k", "v", "slope") if s[n] is not None]
    grads = torch.autograd.grad(out, [s[n] for n in wrt], s["dout"])
    return {"out": out.detach(), **{"d" + n: g for n, g in zip(wrt, grads)}}


def _own_step(s):
    from dgl_amd.attention import PagedCache, attention_step
    cache = PagedCache.over(s["k_pages"], s["v_pages"], s["table"], s["lengths"])
    if s["k_new"] is not None:
        cache.append(s["k_new"], s["v_new"], start=s["start"])
    out = attention_step(s["q"], cache, rows_per_instance=s["rows"], scale=s["scale"], cap=s["cap"], slope=s["slope"],
                         pos_q=s["pos_q"], pos_k=s["pos_k"], blocked=s["blocked"])
    return {"out": out, "k_pages": cache.k_pages, "v_pages": cache.v_pages} if s["k_new"] is not None else {"out": out}


def _own_logits(s):
    from dgl_amd.logits import process_logits
    penalties = s["repetition"] is not None and s["history"] is not None
    log_probs, selected = process_logits(
        s["logits"], blocked=s["blocked"], period=s["period"], bias=s["bias"], temperature=s["temperature"],
        history=s["history"] if penalties else None, history_len=s["history_len"] if penalties else None,
        repetition=s["repetition"] if penalties else 1.0, presence=s["presence"] if penalties else 0.0,
        frequency=s["frequency"] if penalties else 0.0)
    return {"log_probs": log_probs, "selected": selected}


def run(state):
    if own:
        return {"attention": _own_attention, "step": _own_step, "logits": _own_logits}[state["op"]](state)
    return {"attention": _plain_attention, "step": _plain_step, "logits": _plain_logits}[state["op"]](state)


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "logits":
        n = case["rows"] * case["actions"]
        size = 4 if case["dtype"] == "f32" else 2
        bias = 0 if case["bias"] == "none" else 4 * case["actions"] * (case["rows"] if case["bias"] == "rows" else 1)
        history = 4 * case["rows"] * case["history"] // 2 if case["penalties"] else 0
        bits = case["rows"] * ((case["period"] + 63) // 64) * 8 if case["blocked"] else 0
        return {"bytes": n * (size + 4) + bias + history + bits, "flops": 6 * n}
    size = 4 if case["dtype"] == "f32" else 2
    B, H, K, L, D = (case[n] for n in ("batch", "heads", "kv_heads", "length", "dim"))
    if case["op"] == "step":
        live = L * 3 // 4 if case["ragged"] else L
        share = 0.5 if case["blocked"] else 1.0
        rows = B * case["rows"]
        return {"bytes": 2 * B * live * K * D * size + 2 * rows * H * D * size + (8 * B * L if case["bias"] == "coords" else 0)
                + (rows * ((L + 63) // 64) * 8 if case["blocked"] else 0), "flops": 4 * rows * H * live * D * share}
    M = case["keys"]
    pairs = L * M
    if case["causal"]:
        pairs = min(L, M) * (min(L, M) + 1) // 2 + max(0, M - L) * L
    if case["docs"]:
        pairs = pairs * 2 // (case["docs"] + 1)  # what uniform cuts leave of a square, in the mean
    pairs = max(pairs, 1)
    tensors = B * D * size * (2 * H * L + 2 * K * M)
    coords = 8 * B * (L + M) if case["bias"] == "coords" else 0
    if not case["train"]:
        return {"bytes": tensors + coords, "flops": 4 * B * H * pairs * D}
    return {"bytes": B * D * size * (4 * H * L + 4 * K * M) + coords, "flops": 14 * B * H * pairs * D}


# ------------------------------------------------------------------------------------------------------------- exact
def _exact_pairs(s, b, Lq, Lk):
    """(distance or None, allowed) of batch entry b, in 64 bits."""
    rows = torch.arange(Lq, device=DEV, dtype=torch.float64).view(-1, 1) + float(Lk - Lq)
    cols = torch.arange(Lk, device=DEV, dtype=torch.float64).view(1, -1)
    ok = torch.ones(Lq, Lk, dtype=torch.bool, device=DEV)
    if s["causal"]:
        ok &= cols <= rows
        if s["prefix"] is not None:
            ok |= cols < float(s["prefix"][b])
    if s["doc_q"] is not None:
        ok &= s["doc_q"][b].view(-1, 1) == s["doc_k"][b].view(1, -1)
        ok &= s["doc_k"][b].view(1, -1) >= 0
    if s["slope"] is None:
        return None, ok
    if s["pos_q"] is not None:
        return torch.cdist(s["pos_q"][b].double(), s["pos_k"][b].double(), compute_mode="donot_use_mm_for_euclid_dist"), ok
    return (rows - cols).abs(), ok


def _exact_attention(s):
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    B, H, L, D = q.shape
    K, M = k.shape[1], k.shape[2]
    names = ["out"] + (["dq", "dk", "dv"] + (["dslope"] if s["slope"] is not None else []) if s["train"] else [])
    res = {"out": torch.zeros_like(q), "dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v),
           "dslope": torch.zeros(H, dtype=torch.float64, device=DEV)}
    for b in range(B):
        dist, ok = _exact_pairs(s, b, L, M)
        some = ok.any(1, keepdim=True)
        for h in range(H):
            kh, vh = k[b, h * K // H], v[b, h * K // H]
            u = s["scale"] * (q[b, h] @ kh.t())
            y = u if s["cap"] == 0 else s["cap"] * torch.tanh(u / s["cap"])
            if dist is not None:
                y = torch.addcmul(y, dist, -s["slope"].detach()[h].double())
            y = y.masked_fill(~ok, -math.inf)
            w = torch.exp(y - torch.where(some, torch.logsumexp(y, 1, keepdim=True), torch.zeros((), dtype=torch.float64, device=DEV)))
            o = w @ vh
            res["out"][b, h] = o
            if s["train"]:
                do = s["dout"][b, h].double()
                dy = w * (do @ vh.t() - (do * o).sum(1, keepdim=True))
                if dist is not None:
                    res["dslope"][h] -= (dy * dist).sum()
                du = dy if s["cap"] == 0 else dy / torch.cosh(u / s["cap"]).square()
                res["dq"][b, h] = s["scale"] * (du @ kh)
                res["dk"][b, h * K // H] += s["scale"] * (du.t() @ q[b, h])
                res["dv"][b, h * K // H] += w.t() @ do
    return {n: res[n] for n in names}


def _exact_step(s):
    q = s["q"].double()
    R, H, D = q.shape
    P, page, K = s["rows"], s["page"], s["k_pages"].shape[1]
    out = torch.zeros_like(q)
    kp, vp = s["k_pages"], s["v_pages"]
    for b in range(s["table"].shape[0]):
        n = int(s["lengths"][b])
        if s["k_new"] is not None:
            last, slot = int(s["table"][b, (n - 1) // page]), (n - 1) % page
            kp[last, :, slot], vp[last, :, slot] = s["k_new"][b, :, 0], s["v_new"][b, :, 0]
        ids = s["table"][b].long()
        keys = torch.cat(list(kp[ids]), 1)[:, :n].double()
        values = torch.cat(list(vp[ids]), 1)[:, :n].double()
        where = torch.arange(n, device=DEV)
        free = torch.ones(P, n, dtype=torch.bool, device=DEV)
        if s["blocked"] is not None:
            words = s["blocked"][b * P:(b + 1) * P]
            free = ((words[:, where // 64] >> (where % 64)) % 2) == 0
        dist = None
        if s["slope"] is not None:
            dist = (float(n - 1) - where.double()).abs().expand(P, n) if s["pos_q"] is None else torch.cdist(
                s["pos_q"][b * P:(b + 1) * P].double(), s["pos_k"][b, :n].double(), compute_mode="donot_use_mm_for_euclid_dist")
        for h in range(H):
            y = s["scale"] * (q[b * P:(b + 1) * P, h] @ keys[h * K // H].t())
            if s["cap"] > 0:
                y = s["cap"] * torch.tanh(y / s["cap"])
            if dist is not None:
                y = y - s["slope"][h].double() * dist
            w = torch.softmax(y.masked_fill(~free, -math.inf), 1).nan_to_num(0.0)
            out[b * P:(b + 1) * P, h] = w @ values[h * K // H]
    return {"out": out, "k_pages": kp.double(), "v_pages": vp.double()} if s["k_new"] is not None else {"out": out}


def _exact_logits(s):
    x = s["logits"].double()
    R, A = x.shape
    if s["history"] is not None and s["repetition"] is not None:
        seen = torch.zeros(R * A, dtype=torch.float64, device=DEV)
        live = torch.arange(s["history"].shape[1], device=DEV)[None] < s["history_len"][:, None]
        flat = (torch.arange(R, device=DEV)[:, None] * A + s["history"])[live]
        seen.index_add_(0, flat, torch.ones_like(flat, dtype=torch.float64))
        seen = seen.view(R, A)
        r, a, f = (s[n].double().view(R, 1) for n in ("repetition", "presence", "frequency"))
        x = torch.where(seen > 0, x * r ** -torch.sign(x) - a - f * seen, x)
    if s["bias"] is not None:
        x = x + s["bias"].double()
    x = x / float(torch.tensor(s["temperature"], dtype=torch.float32))
    if s["blocked"] is not None:
        col = torch.arange(A, device=DEV) % s["period"]
        x = x.masked_fill(((s["blocked"][:, col // 64] >> (col % 64)) % 2) != 0, -math.inf)
    lp = torch.log_softmax(x, 1)
    return {"log_probs": torch.where(torch.isinf(x), torch.full_like(x, -math.inf), lp), "selected": None}


def exact(case, seed):
    if case["op"] == "attention" and case["batch"] * case["heads"] * case["length"] * case["keys"] > 4e9:
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "step": _exact_step, "logits": _exact_logits}[case["op"]](s)
