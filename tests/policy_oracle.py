"""The policy operators' definitions in 64 bits (plain torch, on the device of the logits), and how far f32 kernels may be off.

Units: h = 2^-24, half a step of f32.  A row's sum of V exponentials, each thread adding at most V / 64 of
them before a tree, is off by at most (V / 64 + 16) h of itself; an exponential 2^u by its instruction's 2 h and by
its argument's rounding (two operations and the rounded factor log2(e) / T, 4 h |u|); `slack` adds
these.  A result in the logits' type is rounded once more: eps / 2."""
import math

import torch

H = 2.0 ** -24
# the exponential's instruction returns 0 for results under the smallest normal number, 2^-126, and what it is given is
# 2^u = p s with s >= 2^-0.5 (the reference is the maximum's, rounded to a whole number): a probability below 2^-125.5 may
# be 0, which moves a gradient by at most that times its factor (no sum of 2^30 such terms reaches h times a sum >= 1)
FLUSHED = 2.0 ** -125.5
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def softmax64(x, mask, T):
    """x [n, V] any type -> z = x / T (illegal: -inf), lse, logp, p in f64; a row without a legal action: p = 0"""
    z = x.detach().double() / T
    if mask is not None:
        z = torch.where(mask.to(x.device).bool(), z, torch.full_like(z, -math.inf))
    m = z.max(1, keepdim=True).values
    none = m[:, 0] == -math.inf
    # from the maximum, not from lse: next to the type's lowest value the logarithm of the sum is lost even in f64
    ln = (z - m).exp().sum(1).log()
    lse = torch.where(none, m[:, 0], m[:, 0] + ln)
    logp = torch.where(none[:, None], torch.full_like(z, -math.inf), (z - m) - ln[:, None])
    return z, lse, logp, torch.where(none[:, None], torch.zeros_like(z), logp.exp())


def row_slack(z, p):
    """[n]: how far ln(sum) and with it every log-probability may be off, beside 3 h |z - max|"""
    V = z.shape[1]
    m = z.max(1, keepdim=True).values
    u = torch.where(torch.isfinite(z), (m - z) / math.log(2.0), torch.zeros_like(z))
    u = torch.where(torch.isfinite(u), u, torch.zeros_like(u))
    eu = (p * u).sum(1)  # mean |u|
    return H * (V / 64 + 40 + 4 * eu + 2 * torch.log1p((z > -math.inf).sum(1).double())), eu


def logprobs(x, actions, mask, T, top):
    """dict of f64 results and their tolerances"""
    n, V = x.shape
    z, lse, logp, p = softmax64(x, mask, T)
    none = lse == -math.inf
    ent = -torch.special.xlogy(p, p).sum(1)
    sl, eu = row_slack(z, p)
    m = z.max(1).values
    r = {"lse": (lse, sl + 3 * H * m.abs().nan_to_num(0, 0, 0)), "entropy": (ent, 2 * sl * (2 + eu))}
    if actions is not None:
        a = actions.to(x.device).long().reshape(-1)
        inside = (a >= 0) & (a < V)
        la = logp.gather(1, a.clamp(0, V - 1)[:, None])[:, 0]
        la = torch.where(inside, la, torch.zeros_like(la))
        za = (z.gather(1, a.clamp(0, V - 1)[:, None])[:, 0] - m).abs().nan_to_num(0, 0, 0)
        r["logp"] = (la, sl + 4 * H * za)
    if top:
        key = x.detach().float()
        key = torch.where(torch.isfinite(z) | (z == math.inf), key, torch.full_like(key, -math.inf))
        v, i = torch.sort(key, dim=1, descending=True, stable=True)
        v, i = v[:, :top], i[:, :top]
        gone = (v == -math.inf) | none[:, None]
        r["top_ids"] = torch.where(gone, torch.full_like(i, -1), i)
        lt = torch.gather(logp, 1, i)
        r["top_logp"] = (torch.where(gone, torch.full_like(lt, -math.inf), lt),
                         sl[:, None] + 4 * H * (torch.gather(z, 1, i) - m[:, None]).abs().nan_to_num(0, 0, 0))
    return r


def logprobs_grad(x, actions, mask, T, g1, g2, g3):
    """(gradient, tolerance) in f64 [n, V]; g1, g2, g3 [n] on logp, entropy, lse"""
    n, V = x.shape
    z, lse, logp, p = softmax64(x, mask, T)
    ent = -torch.special.xlogy(p, p).sum(1, keepdim=True)
    sl, eu = row_slack(z, p)
    g1, g2, g3 = (torch.zeros(n, 1, dtype=torch.float64, device=x.device) if g is None else
                  g.to(x.device).double().reshape(n, 1)
                  for g in (g1, g2, g3))
    hot = torch.zeros(n, V, dtype=torch.float64, device=x.device)
    if actions is not None:
        a = actions.to(x.device).long().reshape(-1)
        inside = (a >= 0) & (a < V) & (lse > -math.inf)
        if mask is not None:
            inside &= mask.to(x.device).bool().gather(1, a.clamp(0, V - 1)[:, None])[:, 0]
        given = (a >= 0) & (a < V)
        hot.scatter_(1, a.clamp(0, V - 1)[:, None], inside.double()[:, None])
        g1 = torch.where(given[:, None], g1, torch.zeros_like(g1))
    lp = torch.where(p > 0, logp, torch.zeros_like(logp))
    d = (g1 * (hot - p) + g3 * p - g2 * p * (lp + ent)) / T
    size = (g1.abs() + g3.abs() + g2.abs() * (ent + lp.abs() + 1)) / T
    eps = torch.finfo(x.dtype).eps
    tol = FLUSHED * size + p * size * (6 * sl[:, None] * (2 + eu[:, None]) + 8 * H * (lp.abs() + 4)) + 4 * H * hot * g1.abs() / T
    return d, tol + eps / 2 * (d.abs() + tol) + TINY[x.dtype]


def distill(x, t_logp, t_ids, mask, T, rest):
    """f64: row losses and their tolerances, the gradient of their sum and its tolerances"""
    n, V = x.shape
    k = t_ids.shape[1]
    z, lse, logp, p = softmax64(x, mask, T)
    sl, eu = row_slack(z, p)
    t = t_logp.detach().to(x.device).double()
    ids = t_ids.to(x.device).long()
    there = (ids >= 0) & (ids < V) & (t != -math.inf)
    ids = ids.clamp(0, V - 1)
    if rest:
        lq = t
    else:
        lq = t - torch.logsumexp(torch.where(there, t, torch.full_like(t, -math.inf)), 1, keepdim=True)
    q = torch.where(there, lq.exp(), torch.zeros_like(t))
    lp = torch.gather(logp, 1, ids)
    term = torch.where(q > 0, q * (lq - lp), torch.zeros_like(q))
    loss = term.sum(1)
    # q: expf's 2 h, the division's, its argument's rounding; the student's logarithm: sl and 3 h |z - max|
    dq = q * 8 * H
    m = z.max(1, keepdim=True).values
    zj = (torch.gather(z, 1, ids) - m).abs().nan_to_num(0, 0, 0)
    tol = (q * (sl[:, None] + 4 * H * zj) + dq * ((lq - lp).abs().nan_to_num(0, 0, 0) + 1)).where(
        there, torch.zeros_like(q)).sum(1)
    tgt = torch.zeros_like(z).scatter_add_(1, ids, q)
    inside = torch.zeros_like(z).scatter_add_(1, ids, there.double()) > 0
    S = q.sum(1)
    dS = dq.sum(1)
    rp = torch.zeros_like(p)
    dr = torch.zeros_like(p)
    if rest:
        out = (z > -math.inf) & ~inside
        lpr = torch.logsumexp(torch.where(out, logp, torch.full_like(logp, -math.inf)), 1)
        qr = (1 - S).clamp_min(0)
        has = (qr > 0) & (lpr > -math.inf)
        # 1 - sum q is off by dS also where it comes out as 0 or below
        may = (1 - S + dS > 0) & (lpr > -math.inf)
        qr = torch.where(has, qr, torch.zeros_like(qr))
        lr = torch.where(has, lpr, torch.zeros_like(lpr))
        lqr = torch.where(has, qr, torch.ones_like(qr)).log()
        loss = loss + qr * (lqr - lr)
        lr = torch.where(may, lpr, torch.zeros_like(lpr))
        lqm = torch.maximum(qr, dS).clamp_min(1e-300).log()
        tol = tol + torch.where(may, dS * ((lqr - lr).abs() + (lqm - lr).abs() + 1) + qr * (2 * sl + 8 * H * lr.abs()),
                                dS * 0)
        S = S + qr
        # p / p_R by the outside's own maximum: p and p_R may both be 0 in f64
        zo = torch.where(out, z, torch.full_like(z, -math.inf))
        zo = zo - torch.where(may[:, None], zo.max(1, keepdim=True).values, torch.zeros_like(lr)[:, None])
        eo = torch.where(out & may[:, None], zo.exp(), torch.zeros_like(p))
        so = eo.sum(1, keepdim=True).clamp_min(1e-300)
        po = eo / so
        rp = torch.where(has[:, None], po * qr[:, None], torch.zeros_like(p))
        lpo = torch.where(po > 0, zo - so.log(), torch.zeros_like(p)).abs()
        # p' has its own sum (its mean |u| beside that of sl) and its own logarithm
        dr = po * dS[:, None] + rp * (3 * sl[:, None] + 8 * H * (lpo + 2) + 12 * H * (po * lpo).sum(1, keepdim=True))
    nothing = (lse == -math.inf) | ~there.any(1)
    loss = torch.where(nothing, torch.zeros_like(loss), loss)
    tol = tol + H * loss.abs().nan_to_num(0, 0, 0)
    if mask is not None:
        tgt = torch.where(mask.to(x.device).bool(), tgt, torch.zeros_like(tgt))
    d = torch.where(nothing[:, None], torch.zeros_like(p), (p * S[:, None] - tgt - rp) / T)
    lpa = torch.where(p > 0, logp, torch.zeros_like(p)).abs()
    dd = p * S[:, None] * (3 * sl[:, None] + 8 * H * (lpa + 2)) + p * dS[:, None] + 16 * H * tgt + dr + FLUSHED * (1 + S[:, None])
    return loss, tol, d, dd / T


def grad_tol(d, dd, w, dtype):
    """tolerance of w d rounded to dtype, dd that of d"""
    t = dd * w.abs() + 4 * H * (d * w).abs()
    return t + torch.finfo(dtype).eps / 2 * ((d * w).abs() + t) + TINY[dtype]


def check(got, want, tol, what):
    most = torch.finfo(got.dtype).max
    got = got.detach().double().reshape(want.shape)
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    same |= torch.isinf(got) & (got * want > 0) & (want.abs() > most)  # beyond the type's largest number
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    bad = ~(same | (off <= tol))
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at "
                           f"{tuple(int(i) for i in bad.nonzero()[0])}: got {got[bad][0]!r}, want {want[bad][0]!r}, "
                           f"tolerance {tol.expand_as(want)[bad][0]!r}")
