"""Attention with its gradients in 64 bits, term by term from the definition, and how far a kernel may be from it.

The bounds follow the operator's arithmetic: binary32 products, scores and sums (unit roundoff u = 2^-24), for 16-bit
types a rounding of probabilities and score gradients before the second product, of the stored output (whose rounding
reaches delta = dout.out) and of the results (half a step, finfo.eps / 2 relative).  With S_ij = |scale| sum_d |q_id k_jd|
the score's error is at most u (D + 8) S_ij + u (16 cap + 16 |s_ij|) (dot product; tanh to 4 ulp, bias and the change to
base 2), which goes into p twice (own score, the row's sum); a sum of n terms adds u n at the most, so u (64 + n) covers
the online rescaling.  For half precision 2^-24 is the spacing near zero: absolute terms follow from the scalings."""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else U


def allowed_pairs(B, Lq, Lk, causal, prefix, doc_q, doc_k, device):
    i = torch.arange(Lq, device=device)[:, None] + (Lk - Lq)
    j = torch.arange(Lk, device=device)[None]
    ok = torch.ones(B, Lq, Lk, dtype=torch.bool, device=device)
    if causal:
        ok = ok & (j <= i)[None]
        if prefix is not None:
            ok = ok | (j[None] < prefix.view(B, 1, 1))
    if doc_q is not None:
        ok = ok & (doc_q[:, :, None] == doc_k[:, None, :]) & (doc_k >= 0)[:, None, :]
    return ok


def reference(q, k, v, dout=None, scale=None, cap=0.0, slope=None, pos_q=None, pos_k=None, doc_q=None, doc_k=None,
              causal=False, prefix=None):
    """Values and bounds: {"out": (value, bound), ...}.  Masked pairs are taken out before anything is multiplied."""
    dtype = q.dtype
    B, H, L, D = q.shape
    K, M = k.shape[1], k.shape[2]
    G = H // K
    scale = D ** -0.5 if scale is None else scale
    ok = allowed_pairs(B, L, M, causal, prefix, doc_q, doc_k, q.device)[:, None]
    # operands of rows that no allowed pair touches may hold anything: they are zero here
    rows, cols = ok.any(-1)[..., None], ok.any(-2)[..., None]
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    qd = torch.where(rows, q.double(), zero)
    kd = torch.where(cols, k.double(), zero).repeat_interleave(G, 1)
    vd = torch.where(cols, v.double(), zero).repeat_interleave(G, 1)
    ok = ok.expand(B, H, L, M)
    x = scale * (qd @ kd.transpose(2, 3))
    S = abs(scale) * (qd.abs() @ kd.abs().transpose(2, 3))
    th = torch.tanh(x / cap) if cap > 0 else torch.zeros_like(x)
    s = cap * th if cap > 0 else x
    dist = torch.zeros_like(x)
    if slope is not None:
        if pos_q is not None:
            d = pos_q.double()[:, :, None] - pos_k.double()[:, None]
            d = d.square().sum(-1).sqrt()[:, None]
        else:
            d = ((torch.arange(L, device=q.device)[:, None] + (M - L)) - torch.arange(M, device=q.device)[None]).abs().double()
        dist = d.expand(B, H, L, M).nan_to_num(0.0)
        s = s - slope.double().view(1, H, 1, 1) * dist
    err_s = U * ((D + 8) * S + 16 * cap + 16 * s.abs())
    if slope is not None:
        err_s = err_s + 8 * U * slope.double().abs().view(1, H, 1, 1) * dist
    s = torch.where(ok, s, -math.inf)
    m = s.amax(-1, keepdim=True) if M else torch.full((B, H, L, 1), -math.inf, dtype=torch.float64, device=q.device)
    live = m > -math.inf
    e = torch.exp(s - torch.where(live, m, zero))
    l = e.sum(-1, keepdim=True)
    p = torch.where(live, e / torch.where(live, l, zero + 1), zero)
    err_s = torch.where(ok, err_s, zero)
    worst = err_s.amax(-1, keepdim=True) if M else torch.zeros_like(m)
    h = 0.0 if dtype == torch.float32 else half_step(dtype)
    rel_p = err_s + worst + U * (64 + M)
    out = p @ vd
    res = {"out": (out, (p * (rel_p + h)) @ vd.abs() + half_step(dtype) * out.abs() * 1.01 + 1e-30)}
    if dtype == torch.float16:   # probabilities relative to the running maximum keep 2^-25 absolutely
        res["out"] = (out, res["out"][1] + 2.0 ** -25 * (ok.double() @ vd.abs()) / torch.where(live, l, zero + 1) + 2.0 ** -25)
    lse = torch.where(live, torch.where(live, m, zero) + torch.log(torch.where(live, l, zero + 1)), -math.inf)[..., 0]
    res["lse"] = (lse, worst[..., 0] * 1.01 + U * (64 + M) + 4 * U * lse.abs().nan_to_num(0, 0, 0))
    if dout is None:
        return res
    do = torch.where(rows, dout.double(), zero)
    dp = do @ vd.transpose(2, 3)
    delta = (do * out).sum(-1, keepdim=True)
    err_dp = U * (D + 2) * (do.abs() @ vd.abs().transpose(2, 3))
    # with the exact softmax the rounding of out reaches delta; the kernels' own error of out does as well
    err_delta = (do.abs() * res["out"][1]).sum(-1, keepdim=True) + U * (D + 2) * (do.abs() * out.abs()).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    err_ds = p * (err_dp + err_delta) + (rel_p + 2 * U) * ds.abs()
    slack = 1 - th * th if cap > 0 else torch.ones_like(ds)
    err_slack = (32 * U + 2 * U * (D + 8) * S / cap) if cap > 0 else 0.0     # of 1 - tanh^2, absolute
    du = ds * slack
    err_du = err_ds * slack + ds.abs() * err_slack + h * du.abs() + 2 * U * du.abs()
    if dtype == torch.float16:   # scaled by the row's (block's) largest gradient: an absolute 2^-25 of that scale's 1/8
        top = do.abs().amax() / 4
        err_du = err_du + torch.where(ok, 2.0 ** -25 * top, zero)
        err_p16 = torch.where(ok, zero + 2.0 ** -35, zero)
    else:
        err_p16 = zero
    n = U * 64
    hs = half_step(dtype)
    fold = lambda t: t.view(B, K, G, M, D).sum(2)  # noqa: E731
    dq = scale * (du @ kd)
    dk = fold(scale * (du.transpose(2, 3) @ qd))
    dv = fold(p.transpose(2, 3) @ do)
    res["dq"] = (dq, abs(scale) * ((err_du + (n + U * M) * du.abs()) @ kd.abs()) + 1.01 * hs * dq.abs())
    res["dk"] = (dk, fold(abs(scale) * ((err_du + (n + U * G * L) * du.abs()).transpose(2, 3) @ qd.abs())) + 1.01 * hs * dk.abs())
    err_p = p * (rel_p + h + n + U * G * L) + err_p16
    res["dv"] = (dv, fold(err_p.transpose(2, 3) @ do.abs()) + 1.01 * hs * dv.abs())
    if dtype == torch.float16:
        for name in ("dq", "dk", "dv"):
            res[name] = (res[name][0], res[name][1] + 2.0 ** -24)
    if slope is not None:
        dslope = -(ds * dist).sum((0, 2, 3))
        # delta's error drops out here (sum_j ds_ij is made zero), to first order
        e = (p * err_dp + (rel_p + 2 * U) * ds.abs() + 8 * U * ds.abs()) * dist + U * (64 + M) * p * (dp.abs() + delta.abs()) * dist
        e = e + p * (p * (err_dp + U * dp.abs())).sum(-1, keepdim=True) * dist + U * p * err_delta * dist * M
        res["dslope"] = (dslope, e.sum((0, 2, 3)) + U * (64 + L) * (ds.abs() * dist).sum((0, 2, 3)) + 1e-30)
    return res


def assert_within(got, want, what):
    value, bound = want
    got = got.double()
    assert got.shape == value.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(value.shape)}"
    inf = torch.isinf(value)
    assert torch.equal(torch.isinf(got) & ~torch.isnan(got), inf), f"{what}: infinities differ"
    off = torch.where(inf, torch.zeros_like(value), (got - value).abs())
    bad = ~(off <= bound)
    if bad.any():
        at = int((off / bound.clamp_min(1e-300)).nan_to_num(math.inf).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off; worst at {at}: got {got.flatten()[at]:.9g}, "
                             f"expected {value.flatten()[at]:.9g} within {bound.flatten()[at]:.3g}")
