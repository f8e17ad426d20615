"""The operators together, as a solver uses them: controls on the policy's rollouts, and a decoder that attends over all
unvisited nodes of cached instances and picks by processed logits."""
import math

import pytest
import torch

from attention_reference import assert_within, reference

pytestmark = pytest.mark.gpu


def tsp(device, B=6, N=40, rpi=1, knn=20, seed=0, weights="trained"):
    import os
    from conftest import GOLDEN
    from dgl_amd._lib import PROBLEM_TSP
    from dgl_amd.engine import PackedPolicy, TspEngine
    from dgl_amd.weights import load_checkpoint
    from oracle.dgl_oracle import random_weights
    g = torch.Generator().manual_seed(seed)
    eng = TspEngine(torch.rand(B, N, 2, generator=g).to(device), rpi, knn)
    sd = load_checkpoint(os.path.join(GOLDEN, "ckpt_tsp_nn.pt")) if weights == "trained" else random_weights("TSP", 3)
    return eng, PackedPolicy(sd, PROBLEM_TSP, device), torch.full((B * rpi,), 3, dtype=torch.int32, device=device)


def cvrp(device, B=5, N=30, rpi=1, knn=10, weights="trained"):
    import os
    from conftest import GOLDEN
    from dgl_amd._lib import PROBLEM_CVRP
    from dgl_amd.engine import CvrpEngine, PackedPolicy
    from dgl_amd.weights import load_checkpoint
    from oracle.dgl_oracle import random_weights
    g = torch.Generator().manual_seed(5)
    xy = torch.rand(B, N + 1, 2, generator=g).to(device)
    dem = torch.cat((torch.zeros(B, 1), torch.randint(1, 200, (B, N), generator=g) / 500.0), 1).to(device)
    eng = CvrpEngine(xy, dem, rpi, knn, knn)
    sd = load_checkpoint(os.path.join(GOLDEN, "ckpt_cvrp_nn.pt")) if weights == "trained" else random_weights("CVRP", 3)
    return eng, PackedPolicy(sd, PROBLEM_CVRP, device), torch.full((B * rpi,), 2 + N + 4, dtype=torch.int32, device=device)


def assert_tours(t, N, first=0):
    assert torch.equal(t.long().sort(1)[0], torch.arange(first, N + first, device=t.device).expand(t.shape[0], N))


def test_controls_that_change_nothing(device):
    from dgl_amd.logits import LogitControls
    for make in (tsp, cvrp):
        eng, pol, start = make(device)
        plain = eng.greedy_rollout(pol, start).clone()
        tours = eng.state["tour" if make is tsp else "nodes"].clone()
        same = eng.greedy_rollout(pol, start, controls=LogitControls())
        assert torch.equal(same, plain) and torch.equal(eng.state["tour" if make is tsp else "nodes"], tours)
        eng, pol, start = make(device, rpi=4)
        plain = eng.beam_rollout(pol, start, 4).view(-1, 4).amin(1).clone()
        same = eng.beam_rollout(pol, start, 4, controls=LogitControls()).view(-1, 4).amin(1)
        # the log-softmax renormalises by the floors' sum: scores move by 1e-6, and only a tie that close may turn
        assert int((same != plain).sum()) <= 1


def test_bias_blocks_and_temperature_steer_a_rollout(device):
    from dgl_amd.logits import LogitControls
    N = 20
    eng, pol, start = tsp(device, N=N, knn=N - 1, weights="random")
    bias = torch.zeros(N, device=device)
    bias[7] = -60.0
    eng.greedy_rollout(pol, start, controls=LogitControls(bias=bias))
    assert (eng.state["tour"][:, -1] == 7).all() and (eng.state["tour"] == 7).sum() == eng.R
    blocked = torch.zeros(eng.R, 1, dtype=torch.int64, device=device)
    blocked[:] = (1 << 5) | (1 << 11)                     # taken when nothing else is left
    eng.greedy_rollout(pol, start, controls=LogitControls(blocked=blocked))
    assert set(eng.state["tour"][:, -2:].flatten().tolist()) == {5, 11}
    first = torch.full((eng.R, 1), 12, dtype=torch.int32, device=device)   # penalised: not the next node
    eng.greedy_rollout(pol, start, controls=LogitControls(history=first, presence=30.0))
    assert (eng.state["tour"][:, -1] == 12).all()
    eng, pol, start = tsp(device, rpi=4)
    length = eng.beam_rollout(pol, start, 4, controls=LogitControls(temperature=2.0))
    best = length.view(-1, 4).argmin(1)
    assert_tours(eng.state["tour"].view(-1, 4, eng.N)[torch.arange(len(best), device=device), best], eng.N)


def test_cvrp_controls_keep_capacity(device):
    """Infeasible moves stay out however the controls push them."""
    from dgl_amd.logits import LogitControls
    eng, pol, start = cvrp(device, weights="random")
    N = eng.N
    bias = torch.zeros(2 * (N + 1), device=device)
    bias[:N + 1] = 40.0                                   # never return to the depot unless it is the only way
    eng.greedy_rollout(pol, start, controls=LogitControls(bias=bias, temperature=3.0))
    assert_tours(eng.state["nodes"], N, 1)
    assert (eng.state["capacity"] >= -1e-5).all()
    load = torch.zeros(eng.R, device=device)
    for t in range(N):
        d = eng.demand.gather(1, eng.state["nodes"][:, t:t + 1].long())[:, 0]
        load = torch.where(eng.state["flags"][:, t] == 1, d, load + d)
        assert (load <= 1 + 1e-5).all()


def test_tester_takes_controls(device):
    from dgl_amd import TSPTester
    from dgl_amd.logits import LogitControls
    import os
    from conftest import GOLDEN
    tp = {"use_cuda": True, "cuda_device_num": 0, "knn": 20, "test_batch_size": 4, "beam_size": 1, "problem_size": 30,
          "test_episodes": 4, "test_episodes_all": 4, "model_load": {"enable": True, "path": GOLDEN, "file": "ckpt_tsp_nn.pt"}}
    import tempfile
    from dgl_amd import formats
    with tempfile.TemporaryDirectory() as d:
        path = os.path.join(d, "x.txt")
        formats.write_tsp_instances(path, torch.rand(4, 30, 2, generator=torch.Generator().manual_seed(0)))
        env = {"mode": "test", "test_mode": "pomo_test", "aug_size": 1, "data_path": path, "baseline_path": ""}
        model = {"mode": "test", "embedding_dim": 128, "head_num": 8, "qkv_dim": 16, "ff_hidden_dim": 512, "decoder_layer_num": 3}
        scores = []
        for extra in ({}, {"logit_controls": LogitControls()}):
            t = TSPTester(env_params=dict(env), model_params=dict(model), tester_params=dict(tp, **extra))
            t.run()
            scores.append(t.score)
        assert scores[0] == scores[1]
        t = TSPTester(env_params=dict(env), model_params=dict(model),
                      tester_params=dict(tp, logit_controls=LogitControls(), reference_protocol=True))
        with pytest.raises(ValueError, match="logit_controls"):
            t.run()


def encoder(xy, H, D, seed):
    """Random linear maps of the coordinates and a constant to queries, keys and values [B, H, N, D]."""
    g = torch.Generator(device=xy.device).manual_seed(seed)
    x = torch.cat((xy, torch.ones_like(xy[..., :1])), -1)
    out = []
    for _ in range(3):
        w = torch.randn(3, H * D, device=xy.device, generator=g)
        out.append((x @ w).view(*xy.shape[:2], H, D).transpose(1, 2))
    return out


def test_attention_over_unvisited_nodes_of_the_state(device):
    from dgl_amd.attention import PagedCache
    B, N, rpi, H, D = 3, 100, 4, 8, 16
    eng, pol, start = tsp(device, B=B, N=N, rpi=rpi)
    q, k, v = encoder(eng.xy, H, D, 1)
    cache = PagedCache(B, H, D, N, device=device)
    cache.append(k, v)
    slope = torch.rand(H, device=device)
    eng.reset()
    seq = torch.arange(eng.R, device=device) // rpi
    pick = torch.stack([torch.randperm(N, generator=torch.Generator().manual_seed(r)) for r in range(eng.R)]).to(device)
    for t in range(N):
        eng.step(pick[:, t].to(torch.int32))
        if t not in (0, 1, 50, 98, 99):
            continue
        rows = q[seq, :, pick[:, t]].contiguous()
        got = eng.attend(rows, cache, cap=10.0, slope=slope)
        seen = torch.zeros(eng.R, N, dtype=torch.int32, device=device).scatter_(1, pick[:, :t + 1], -1)
        cur = eng.xy[seq, pick[:, t]]
        want = reference(rows[:, :, None], k[seq], v[seq], cap=10.0, slope=slope, pos_q=cur[:, None], pos_k=eng.xy[seq],
                         doc_q=torch.zeros(eng.R, 1, dtype=torch.int32, device=device), doc_k=seen)["out"]
        assert_within(got, (want[0][:, :, 0], want[1][:, :, 0]), f"after {t + 1} nodes")
        if t == N - 1:
            assert not got.any()


def test_a_decoder_of_the_operators(device):
    """Encode once, then per node: attend over the unvisited nodes, score every node against the result, process the
    logits, step the state.  Each decision agrees with the same network in 64 bits up to the margin of its rounding."""
    from dgl_amd.attention import PagedCache, attention
    from dgl_amd.logits import process_logits
    B, N, H, D = 4, 50, 8, 16
    eng, pol, start = tsp(device, B=B, N=N)
    q, k, v = encoder(eng.xy, H, D, 2)
    slope = 1.0 + torch.arange(H, device=device).float()
    enc = attention(q, k, v, cap=10.0, slope=slope, pos_q=eng.xy, pos_k=eng.xy)
    cache = PagedCache(B, H, D, N, page_size=16, device=device)
    cache.append(enc, v)
    keys = enc.transpose(1, 2).reshape(B, N, H * D)
    eng.reset()
    eng.step(start)
    bias = torch.linspace(0, 1, N, device=device)
    rows = torch.arange(B, device=device)
    for t in range(1, N):
        cur = eng.state["tour"][:, t - 1].long()
        ctx = eng.attend(q[rows, :, cur].contiguous(), cache, cap=10.0, slope=slope)
        logits = torch.matmul(keys, ctx.reshape(B, H * D, 1))[..., 0] / math.sqrt(H * D)
        lp, sel = process_logits(logits, blocked=eng.state["visited"], bias=bias, temperature=0.5)
        seen = torch.zeros(B, N, dtype=torch.bool, device=device).scatter_(1, eng.state["tour"][:, :t].long(), True)
        x = ((logits.double() + bias.double()) / 0.5).masked_fill(seen, -math.inf)
        assert torch.isneginf(lp).equal(seen)
        assert (x.amax(1) - x.gather(1, sel.long()[:, None])[:, 0]).abs().max() <= 1e-5 * (1 + x.amax())
        torch.testing.assert_close(lp[~seen].double(), torch.log_softmax(x, 1)[~seen], rtol=1e-5, atol=1e-5)
        eng.step(sel)
    assert_tours(eng.state["tour"], N)


def test_training_and_serving_agree_on_a_causal_encoder(device):
    """Gradients reach the maps that made q, k and v, through autograd."""
    from dgl_amd.attention import attention
    g = torch.Generator(device=device).manual_seed(0)
    x = torch.randn(2, 60, 32, device=device, generator=g)
    w = (torch.randn(32, 3 * 64, device=device, generator=g) * 0.2).requires_grad_(True)
    slope = torch.full((4,), 0.1, device=device, requires_grad=True)
    q, k, v = (x @ w).view(2, 60, 3, 4, 16).permute(2, 0, 3, 1, 4)
    out = attention(q, k, v, causal=True, cap=8.0, slope=slope)
    out.square().sum().backward()
    w64 = w.detach().double().requires_grad_(True)
    s64 = slope.detach().double().requires_grad_(True)
    q, k, v = (x.double() @ w64).view(2, 60, 3, 4, 16).permute(2, 0, 3, 1, 4)
    y = 8.0 * torch.tanh(q @ k.transpose(2, 3) / 4.0 / 8.0)
    i = torch.arange(60, device=device)
    y = y - s64.view(1, 4, 1, 1) * (i[:, None] - i[None]).abs().double()
    y = torch.softmax(y.masked_fill(i[None] > i[:, None], -math.inf), -1) @ v
    y.square().sum().backward()
    for a, b in ((w.grad, w64.grad), (slope.grad, s64.grad)):
        # binary32 products of lengths 60 and 32 before and after the operator: 1e-5 of the gradient's size
        assert float((a.double() - b).norm()) <= 1e-5 * float(b.norm())


@pytest.mark.parametrize("problem", ["tsp", "cvrp"])
def test_attention_between_steps_along_back_pointers(device, problem):
    """The current node of a row after a fused beam step, whose tours are only traced back at the end, and after a plain step
    that follows another rollout."""
    from dgl_amd.attention import PagedCache, attention_step
    B, N, beam, H, D = 3, 30, 4, 4, 16
    eng, pol, start = (tsp if problem == "tsp" else cvrp)(device, B=B, N=N, rpi=beam)
    nodes = eng.xy.shape[1]
    q, k, v = encoder(eng.xy, H, D, 3)
    cache = PagedCache(B, H, D, nodes, page_size=16, device=device)
    cache.append(k, v)
    slope = 1.0 + torch.rand(H, device=device)
    rows = torch.randn(eng.R, H, D, device=device)
    seq = torch.arange(eng.R, device=device) // beam
    at = {"node": start.long() if problem == "tsp" else start.long() - (N + 1)}

    def check_attend():
        want = attention_step(rows, cache, rows_per_instance=beam, slope=slope, pos_q=eng.xy[seq, at["node"]], pos_k=eng.xy,
                              blocked=eng.state["visited"])
        assert torch.equal(eng.attend(rows, cache, slope=slope), want)
    eng.reset()
    eng.step(start)
    check_attend()
    scores = torch.zeros(B, beam, device=device)
    prev_k, action = (torch.zeros(B, beam, dtype=torch.int32, device=device) for _ in range(2))
    for t in range(1, 6):
        eng.forward(pol, want_logits=False)
        eng.beam_advance(scores, beam, t, prev_k, action)
        eng.step_beam(prev_k.view(-1), action.view(-1), beam)
        chosen = action.view(-1).long()
        at["node"] = torch.where(chosen > N, chosen - (N + 1), chosen) if problem == "cvrp" else chosen
        check_attend()
    eng.reset()
    eng.step(start)
    at["node"] = start.long() if problem == "tsp" else start.long() - (N + 1)
    check_attend()
