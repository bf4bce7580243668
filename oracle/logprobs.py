"""CPU oracle (test infra) of token log probabilities, entropy and top
alternatives of rows of logits and their gradient, in 64 bits, row by row."""
import numpy as np


def forward(x, tokens, top):
    """x [rows, V] float64 -> logprob, entropy [rows], ids, top_logprobs [rows, top]."""
    rows, V = x.shape
    lp, ent = np.zeros(rows), np.zeros(rows)
    ids, tlp = np.zeros((rows, top), np.int64), np.zeros((rows, top))
    for r in range(rows):
        logp = row_logp(x[r])
        p = np.exp(logp)
        if 0 <= tokens[r] < V:
            lp[r] = logp[tokens[r]]
        ent[r] = np.nan if np.isnan(logp).any() else -sum(p[p > 0] * logp[p > 0])
        # largest first, equal ones by index, NaN in front
        order = sorted(range(V), key=lambda i: (0 if np.isnan(x[r, i]) else 1, -x[r, i] if x[r, i] == x[r, i] else 0, i))
        ids[r] = order[:top]
        tlp[r] = logp[ids[r]]
    return lp, ent, ids, tlp


def row_logp(x):
    if np.isnan(x).any() or np.isposinf(x).any():
        return np.full_like(x, np.nan)
    if np.isneginf(x).all():
        return x.copy()
    m = x.max()
    return x - m - np.log(np.exp(x - m).sum())


def backward(x, tokens, ids, g_lp=None, g_ent=None, g_top=None):
    """gradient of sum(g_lp lp) + sum(g_ent H) + sum(g_top top_lp) with respect to x."""
    rows, V = x.shape
    dx = np.zeros_like(x)
    for r in range(rows):
        logp = row_logp(x[r])
        if np.isneginf(logp).all():
            continue
        p = np.exp(logp)
        pick = []
        if g_lp is not None and 0 <= tokens[r] < V:
            pick.append((tokens[r], g_lp[r]))
        if g_top is not None:
            pick += list(zip(ids[r], g_top[r]))
        for i, g in pick:
            dx[r] -= g * p
            dx[r, i] += g
        if g_ent is not None:
            plogp = np.where(p > 0, p * np.where(p > 0, logp, 0), 0) if not np.isnan(p).any() else p
            H = -plogp.sum()
            dx[r] -= g_ent[r] * (plogp + p * H)
    return dx
