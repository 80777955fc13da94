"""Plain float64 forms of the serving operators, one request or row at a time."""
import math

import numpy as np
import torch


def ragged(requests):
    """(offsets, lengths) of a list of (new tokens, length)."""
    offsets = [0]
    for n, _ in requests:
        offsets.append(offsets[-1] + n)
    return offsets, [m for _, m in requests]


def rope_tables(length, dim):
    inv = 10000.0 ** (-np.arange(0, dim, 2) / dim)
    angle = np.arange(length)[:, None] * inv[None, :]
    return (torch.from_numpy(np.cos(angle).astype(np.float32)),
            torch.from_numpy(np.sin(angle).astype(np.float32)))


def turn(x, cos, sin):
    """x [tokens, heads, dim] rotated by cos, sin [tokens, dim / 2], in float64."""
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    out = torch.empty_like(x)
    out[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
    out[..., 1::2] = x[..., 0::2] * s + x[..., 1::2] * c
    return out


def attention(q, k, v, first_position):
    """q [n, q_heads, dim] (rotated), k, v [keys, heads, dim], all float64;
    query i stands at first_position + i and sees the keys up to there.
    Returns o, lse, and what the tolerances need: the weighted |v| and the
    largest sum of |q'||k| of a row, scaled."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    o = torch.zeros_like(q)
    weighted = torch.zeros_like(q)
    spread = torch.zeros(n, heads, dtype=torch.float64, device=q.device)
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64, device=q.device)
    at = torch.arange(n, device=q.device) + first_position
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        if kh.shape[0] == 0:
            continue
        hidden = torch.arange(kh.shape[0], device=q.device) > at[:, None]
        s = (q[:, h] @ kh.T / math.sqrt(dim)).masked_fill(hidden, -math.inf)
        some = ~hidden.all(1)
        p = torch.softmax(s[some], 1)
        o[some, h] = p @ vh
        weighted[some, h] = p @ vh.abs()
        lse[some, h] = torch.logsumexp(s[some], 1)
        spread[:, h] = (q[:, h].abs() @ kh.abs().T / math.sqrt(dim)).masked_fill(hidden, 0).amax(1)
    return o, lse, weighted, spread


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(id, log-probability, margin) of one row of logits; margin is the
    distance of the draw from the next border, relative to the total, the
    cuts' borders included."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    if not (x > -np.inf).any():
        return -1, -np.inf, 1.0
    order = np.lexsort((np.arange(x.size), -x))
    if not temperature > 2.0 ** -100:
        return int(order[0]), 0.0, 1.0
    top = x[order[0]]
    if top == np.inf:
        w = (x[order] == np.inf).astype(np.float64)
    else:
        w = np.exp((x[order] - top) / temperature)
    margin = 1.0
    if top_k > 0:
        w[top_k:] = 0.0
    if top_p < 1.0:
        total = w.sum()
        before = np.cumsum(w) - w
        near = np.abs(before[1:][w[1:] > 0] / total - top_p)
        margin = min(margin, near.min() if near.size else 1.0)
        drop = before >= top_p * total
        drop[0] = False
        w[drop] = 0.0
    if min_p > 0.0 and top < np.inf:
        drop = w < min(min_p, 1.0)
        w[drop] = 0.0
    run = np.zeros_like(w)
    run[order] = w
    weights = run.copy()
    run = np.cumsum(run)
    aim = min(max(u, 0.0), 1.0) * run[-1]
    i = int(np.searchsorted(run, aim, side="right"))
    if i >= x.size:
        i = int(np.nonzero(weights)[0][-1])
    else:
        i = i if weights[i] > 0 else int(np.nonzero(weights[i:])[0][0]) + i
    return i, math.log(weights[i] / run[-1]), min(margin, np.abs(run - aim).min() / run[-1])
