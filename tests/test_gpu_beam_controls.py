"""Beam search under controls expands what the policy offers and nothing else, however far the controls push it."""
import math

import pytest
import torch

from test_gpu_search_controls import cvrp, tsp

pytestmark = pytest.mark.gpu


def check_tsp(eng, length):
    """Every row whose length counts is a tour; every group has such a row."""
    fin = length.isfinite()
    tours = eng.state["tour"].long()
    whole = (tours.sort(1)[0] == torch.arange(eng.N, device=tours.device)).all(1)
    assert bool(whole[fin].all()), f"{int((fin & ~whole).sum())} of {len(fin)} rows are no tours and have a length"
    return fin


def check_cvrp(eng, length):
    """... visits every customer once within the capacity."""
    fin = length.isfinite()
    nodes = eng.state["nodes"].long()
    whole = (nodes.sort(1)[0] == torch.arange(1, eng.N + 1, device=nodes.device)).all(1)
    seq = torch.arange(eng.R, device=nodes.device) // eng.rpi
    demand = eng.demand[seq].double().gather(1, nodes)
    load = torch.zeros(eng.R, device=nodes.device, dtype=torch.float64)
    ok = whole.clone()
    for t in range(eng.N):
        load = torch.where(eng.state["flags"][:, t] == 1, demand[:, t], load + demand[:, t])
        ok &= load <= 1 + 1e-5
    assert bool(ok[fin].all()), f"{int((fin & ~ok).sum())} of {len(fin)} rows break the rules and have a length"
    return fin


def controls(kind, R, actions, device):
    from dgl_amd.logits import LogitControls
    if kind == "cold":
        return LogitControls(temperature=0.1)
    if kind == "bias":
        bias = torch.zeros(actions, device=device)
        bias[::2] = -60.0
        return LogitControls(bias=bias)
    if kind == "far bias":
        return LogitControls(bias=torch.where(torch.arange(actions, device=device) % 3 == 0, 0.0, -1e30))
    if kind == "presence":
        every = torch.arange(0, actions, 2, device=device, dtype=torch.int32).expand(R, -1)
        return LogitControls(history=every, presence=200.0)
    blocked = torch.zeros(R, (actions + 63) // 64, dtype=torch.int64, device=device)
    blocked[:, 0] = 0x5555_5555_5555
    return LogitControls(blocked=blocked, temperature=0.3)


KINDS = ["cold", "bias", "far bias", "presence", "blocked"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("knn,beam", [(5, 4), (5, 16), (20, 4), (2, 8)])
def test_tsp_rows_that_count_are_tours(device, kind, knn, beam):
    for weights in ("trained", "random"):
        eng, pol, start = tsp(device, B=4, N=30, rpi=beam, knn=knn, weights=weights)
        length = eng.beam_rollout(pol, start, beam, controls=controls(kind, eng.R, eng.N, device))
        assert bool(check_tsp(eng, length).view(-1, beam).any(1).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("knn,beam", [(4, 4), (4, 16), (10, 4), (1, 8)])
def test_cvrp_rows_that_count_keep_the_rules(device, kind, knn, beam):
    for weights in ("trained", "random"):
        eng, pol, start = cvrp(device, B=4, N=24, rpi=beam, knn=knn, weights=weights)
        length = eng.beam_rollout(pol, start, beam, controls=controls(kind, eng.R, 2 * (eng.N + 1), device))
        assert bool(check_cvrp(eng, length).view(-1, beam).any(1).all())


def test_multi_starts_and_a_rollout_without_controls_afterwards(device):
    from dgl_amd.logits import LogitControls
    eng, pol, start = tsp(device, B=3, N=30, rpi=8, knn=3)
    start = (start + torch.arange(8, device=device).repeat_interleave(4)[: 8].repeat(3)).to(torch.int32)   # two starts of four beams
    length = eng.beam_rollout(pol, start, 4, controls=LogitControls(temperature=0.05))
    assert bool(check_tsp(eng, length).view(-1, 4).any(1).all())
    assert eng.beam_rollout(pol, start, 4).isfinite().all()          # lengths as before without controls


def test_tester_under_augmentation(device):
    """Lengths measured again on the original coordinates keep the rows that do not count out."""
    import os
    import tempfile
    from conftest import GOLDEN
    from dgl_amd import TSPTester, formats
    from dgl_amd.logits import LogitControls
    tp = {"use_cuda": True, "cuda_device_num": 0, "knn": 2, "test_batch_size": 2, "beam_size": 16, "problem_size": 20,
          "test_episodes": 2, "test_episodes_all": 2, "model_load": {"enable": True, "path": GOLDEN, "file": "ckpt_tsp_nn.pt"},
          "logit_controls": LogitControls(temperature=0.1)}
    model = {"mode": "test", "embedding_dim": 128, "head_num": 8, "qkv_dim": 16, "ff_hidden_dim": 512, "decoder_layer_num": 3}
    with tempfile.TemporaryDirectory() as d:
        path = os.path.join(d, "x.txt")
        formats.write_tsp_instances(path, torch.rand(2, 20, 2, generator=torch.Generator().manual_seed(0)))
        for mode, aug in (("pomo_test", 1), ("aug_test", 8)):
            env = {"mode": "test", "test_mode": mode, "aug_size": aug, "data_path": path, "baseline_path": ""}
            t = TSPTester(env_params=env, model_params=dict(model), tester_params=dict(tp))
            t.run()
            assert math.isfinite(t.score)
            fin = t.last_lengths.isfinite()
            whole = (t.last_tours.long().sort(1)[0] == torch.arange(20, device=t.last_tours.device)).all(1)
            assert bool(whole[fin].all())


@pytest.mark.parametrize("problem", ["tsp", "cvrp"])
def test_decisions_offer_candidates_alone(device, problem):
    """One decision: what is above the floor are the policy's feasible candidates, with the softmax of the controlled values."""
    from dgl_amd.engine import controlled_log_probs
    from dgl_amd.logits import LogitControls
    eng, pol, start = (tsp if problem == "tsp" else cvrp)(device, B=6, N=30, knn=7)
    eng.reset()
    eng.step(start)
    for t in range(1, 12):
        eng.forward(pol, want_logits=False)
        bias = torch.randn(eng.N if problem == "tsp" else 2 * (eng.N + 1), device=device) * 40
        lp, sel = controlled_log_probs(eng, LogitControls(bias=bias, temperature=0.2))
        dense = eng.dense_probs().double()
        offered = dense > 1e-19
        if problem == "cvrp":
            near = eng.idx_last[:, :eng.kl].long()
            offered.scatter_(1, near, offered.gather(1, near) & (eng.infeasible[:, :eng.kl] == 0))
        x = torch.where(offered, (dense.log() + bias.double()) / 0.2, -math.inf)
        want = torch.log_softmax(x, 1)
        assert torch.equal(lp > -1e19, offered)
        # binary32: the logarithm, the bias and the division round values of up to 1e3 by 2^-24 each, the sum adds 1e-5
        size = x[offered].abs().max()
        assert (lp.double() - want)[offered].abs().max() <= 8 * 2.0 ** -24 * size + 1e-5
        assert torch.equal(sel.long(), lp.argmax(1))
        eng.step(sel)


@pytest.mark.parametrize("problem", ["tsp", "cvrp"])
def test_improbable_candidates_are_candidates(device, problem):
    """A policy that is certain of one candidate (the others' softmax is below 1e-14, their probability the floor): with that
    one blocked another candidate is taken, not the blocked one."""
    from dgl_amd.logits import LogitControls
    from dgl_amd.engine import PackedPolicy, controlled_log_probs
    eng, pol, start = (tsp if problem == "tsp" else cvrp)(device, B=6, N=30, knn=7, weights="random")
    sd = {n: x.clone() for n, x in pol.sd.items()}
    sd["decoder.Linear_final.weight"] *= 3e4
    pol = PackedPolicy(sd, pol.problem, device)
    eng.reset()
    eng.step(start)
    saw = 0
    for t in range(1, 20):
        eng.forward(pol, want_logits=False)
        own = eng.selected.clone().long()
        near = eng.offered_log_probs()
        offered = near > -math.inf
        alone = (near > math.log(2e-7)).sum(1) == 1                # the rest at the floor
        actions = near.shape[1]
        bits = torch.zeros(eng.R, (actions + 63) // 64, dtype=torch.int64, device=device)
        bits.scatter_(1, (own // 64)[:, None], (torch.ones_like(own) << (own % 64))[:, None])
        lp, sel = controlled_log_probs(eng, LogitControls(blocked=bits))
        more = offered.sum(1) > 1
        assert bool(offered.gather(1, sel.long()[:, None]).all())
        assert bool((sel.long() != own)[more].all()) and bool((sel.long() == own)[~more].all())
        saw += int((alone & more).sum())
        eng.step(sel)
    assert saw > 0


@pytest.mark.parametrize("problem", ["tsp", "cvrp"])
def test_only_candidates_count_for_blocked_actions(device, problem):
    """Small neighbourhoods whose candidates are all blocked: the policy's own choice, though nodes outside are not blocked; and
    a penalty for repetitions multiplies log-probabilities."""
    from dgl_amd.engine import controlled_log_probs
    from dgl_amd.logits import LogitControls
    eng, pol, start = (tsp if problem == "tsp" else cvrp)(device, B=6, N=30, knn=3)
    eng.reset()
    eng.step(start)
    eng.forward(pol, want_logits=False)
    near = eng.offered_log_probs()
    offered = near > -math.inf
    assert bool((offered.sum(1) <= 6).all())
    at = torch.arange(near.shape[1], device=device)
    words = torch.zeros(eng.R, 1, dtype=torch.int64, device=device)
    for r in range(eng.R):
        for a in at[offered[r]].tolist():
            words[r, 0] |= 1 << a if a < 63 else -1 << 63
    lp, sel = controlled_log_probs(eng, LogitControls(blocked=words))
    assert torch.equal(sel, eng.selected) and torch.equal(lp > -1e19, offered)
    best = near.argmax(1)
    lp, _ = controlled_log_probs(eng, LogitControls(history=best.to(torch.int32)[:, None], repetition=3.0))
    x = near.double()
    x.scatter_(1, best[:, None], 3.0 * x.gather(1, best[:, None]))
    assert (lp.double() - torch.log_softmax(x, 1))[offered].abs().max() <= 1e-5
