"""The categorical-policy operators from their definitions, in 64 bits and
row by row or over whole arrays (include/rtenv.h: rt_cat_*), and how far an
f32 kernel may be from them.  Runs on any device; used as the oracle of
tests/test_gpu_categorical.py."""
import math

import numpy as np
import torch

INF = math.inf
UNIT = 2.0 ** 40


def sample_row(x, u, T=1.0, k=0, p=1.0, q=0.0):
    """(action, logprob, kept_logprob) of one row of float64 numbers (numpy)."""
    V = len(x)
    if np.isnan(x).any() or (x == INF).any() or (x == -INF).all():
        return -1, math.nan, math.nan
    m = x.max()
    if not T > 0:
        return int(np.argmax(x)), 0.0, 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(x == -INF, -INF, (x - m) / T)
    w = np.rint(np.exp(z) * UNIT).astype(np.int64)
    order = np.argsort(-x, kind="stable")
    n = V
    if 0 < k < V:
        n = k
    ws = w[order][:n]
    mass = int(ws.sum())
    if p < 1:
        limit = max(1, math.ceil(float(np.float64(np.float32(p)) * np.float64(mass))))
        n = min(n, int((np.cumsum(ws) - ws < limit).sum()))
    keep = np.zeros(V, bool)
    keep[order[:n]] = True
    if q > 0:
        theta = 0.0 if q >= 1 else T * math.log(float(np.float32(q)))
        keep &= x - m >= theta
    run = np.cumsum(np.where(keep, w, 0))
    left = int(run[-1])
    u = min(u, 1.0) if u > 0 else 0.0
    hit = math.floor(float(np.float64(u) * np.float64(left)))
    a = int(np.searchsorted(run, min(hit, left - 1), side="right"))
    return a, float(z[a] - math.log(w.sum() / UNIT)), float(z[a] - math.log(left / UNIT))


def sample(x, u, T, k, p, q):
    """Arrays of sample_row over the rows of x; T, k, p, q: one value per row."""
    got = [sample_row(x[n], float(u[n]), float(T[n]), int(k[n]), float(p[n]), float(q[n])) for n in range(len(x))]
    a, lp, kp = zip(*got)
    return np.array(a), np.array(lp), np.array(kp)


def _softmax(x, T):
    z = x.double() / T
    lp = torch.log_softmax(z, -1)
    p = lp.exp()
    return lp, p, torch.where(p > 0, p * lp, 0.0).sum(-1).neg()


def _counts(x, weights, more):
    """Rows that are not ignored, and their weights."""
    n = x.shape[0]
    w = torch.full((n,), 1.0 / n, dtype=torch.float64, device=x.device) if weights is None else weights.double()
    empty = (x == -INF).all(-1)
    return more & (w != 0) & ~empty, w


def _lse_tol(h):
    # sums of exponentials whose argument is rounded once: sum p |t| 2^-24 ln 2 <= 2^-24 H, each
    # exponential within 2^-23, up to eight added in f32 before they go to 64 bits: 2^-21
    return 2.0 ** -20 * (1 + h)


def _grad_tol(dtype, g, lp, p, h, e, f, named):
    """Per element: the rounding to `dtype` by half a step (and half the least subnormal), and what the
    relative error of p and of the coefficients does (_lse_tol, |lp| 2^-23 of its own argument)."""
    info = torch.finfo(dtype)
    tiny = info.smallest_normal * info.eps
    rel = _lse_tol(h)[:, None] * 2 + lp.abs().clamp(max=200) * 2.0 ** -22
    size = torch.where(p > 0, p * (e[:, None].abs() * (lp.abs().clamp(max=1e30) + 1) + f[:, None].abs()), 0.0) + named.abs()
    return info.eps / 2 * g.abs() + rel * size + tiny


def ppo(x, actions, old, adv, weights=None, ref=None, T=1.0, low=0.2, high=0.2, ent=0.0, klc=0.0, scale=1.0):
    """{name: (value, tolerance)} of rt_cat_ppo on x [n, V]; gradient times `scale`."""
    n, V = x.shape
    live, w = _counts(x, weights, (actions >= 0) & (actions < V))
    xs = torch.where(live[:, None], x, torch.zeros((), dtype=x.dtype, device=x.device))
    a = torch.where(live, actions, 0)
    w = torch.where(live, w, 0.0)
    lps, p, h = _softmax(xs, T)
    lp = lps.gather(1, a[:, None])[:, 0]
    lr = lp - old.double()
    r = lr.exp()
    A = adv.double()
    one, two = -A * r, -A * r.clamp(1 - low, 1 + high)
    pg = torch.maximum(one, two)
    c = torch.where(one >= two, one, 0.0)
    kl = torch.zeros_like(lp)
    away = torch.zeros_like(lp)
    if ref is not None:
        away = ref.double() - lp
        kl = away.exp() - away - 1
        c = c + klc * (1 - away.exp())
    terms = torch.stack([pg, kl, h, -lr, (r - 1) - lr, ((r < 1 - low) | (r > 1 + high)).double()], 1)
    # what an error d of lp does to each term
    d = _lse_tol(h)
    move = torch.stack([one.abs(), (1 - away.exp()).abs(), 2 * (1 + h), torch.ones_like(lp), (r - 1).abs(), torch.zeros_like(lp)], 1)
    stats = torch.where(live[:, None], w[:, None] * terms, 0.0).sum(0)
    stats_tol = torch.where(live[:, None], (w[:, None].abs() * move * d[:, None]), 0.0).sum(0) + stats.abs() * 2.0 ** -24
    loss = stats[0] + klc * stats[1] - ent * stats[2]
    loss_tol = stats_tol[0] + abs(klc) * stats_tol[1] + abs(ent) * stats_tol[2] + loss.abs() * 2.0 ** -24
    E, C = w * ent / T, w * c / T
    F = E * h - C
    delta = torch.zeros_like(p).scatter_(1, a[:, None], 1.0)
    lp0 = torch.where(p > 0, lps, 0.0)
    g = scale * (p * (E[:, None] * lp0 + F[:, None]) + delta * C[:, None])
    g = torch.where(live[:, None], g, 0.0)
    big = w.abs() * (one.abs() + abs(klc) * (1 + away.exp())) / T
    tol = _grad_tol(x.dtype, g, lp0, p, h, scale * E, abs(scale) * (big + (E * h).abs()), abs(scale) * delta * big[:, None])
    z = lambda v: torch.where(live, v, 0.0)  # noqa: E731
    return {"loss": (loss, loss_tol), "stats": (stats, stats_tol), "logprob": (z(lp), z(d + lp.abs() * 2.0 ** -24)),
            "entropy": (z(h), z(2 * d * (1 + h) + h * 2.0 ** -24)), "grad": (g, torch.where(live[:, None], tol, 0.0))}


def distill(x, idx, top, weights=None, lse=None, T=1.0, scale=1.0):
    """{name: (value, tolerance)} of rt_cat_distill."""
    n, V = x.shape
    live, w = _counts(x, weights, torch.ones(n, dtype=torch.bool, device=x.device))
    xs = torch.where(live[:, None], x, torch.zeros((), dtype=x.dtype, device=x.device))
    w = torch.where(live, w, 0.0)
    lps, p, h = _softmax(xs, T)
    there = (idx >= 0) & (idx < V)
    j = torch.where(there, idx, 0)
    t = torch.where(there, top.double() / T, -INF)
    if lse is None:
        norm = torch.logsumexp(t, 1)
        norm = torch.where(norm == -INF, 0.0, norm)
    else:
        norm = lse.double()
    lq = t - norm[:, None]
    q = torch.where(there, lq.exp(), 0.0)
    Q = q.sum(1)
    kl = torch.where(q > 0, q * (lq - lps.gather(1, j)), 0.0).sum(1)
    kl_tol = torch.where(live, Q * _lse_tol(h), 0.0) + kl.abs() * 2.0 ** -24
    kl = torch.where(live, kl, 0.0)
    loss = torch.where(w != 0, w * kl, 0.0).sum()
    named = torch.zeros_like(p).scatter_add_(1, j, w[:, None] / T * q)
    lp0 = torch.where(p > 0, lps, 0.0)
    F = w / T * Q
    g = torch.where(live[:, None], scale * (p * F[:, None] - named), 0.0)
    tol = _grad_tol(x.dtype, g, lp0, p, h, torch.zeros_like(F), abs(scale) * F, abs(scale) * named * 2.0 ** -3)
    return {"loss": (loss, torch.where(w != 0, w.abs() * kl_tol, 0.0).sum() + loss.abs() * 2.0 ** -24), "kl": (kl, kl_tol),
            "grad": (g, torch.where(live[:, None], tol, 0.0))}
