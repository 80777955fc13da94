"""Plain forms of the 8-bit paged cache and of speculative decoding's operators,
written from their definitions."""
import numpy as np
import torch


def e4m3_values():
    """What the 256 bytes of type e4m3 stand for: sign, 4 bits of exponent (bias 7), 3
    of fraction; exponent 0: multiples of 2^-9; 0x7f and 0xff: NaN."""
    b = np.arange(256)
    e, f = (b >> 3) & 15, b & 7
    v = np.where(e > 0, (1 + f / 8.0) * 2.0 ** (e - 7.0), f * 2.0 ** -9.0)
    v[(b & 127) == 127] = np.nan
    return torch.from_numpy(np.where(b >= 128, -v, v))


def rows_of(pool, scales):
    """The float64 rows that bytes [..., dim] and scales [...] stand for."""
    return e4m3_values().to(pool.device)[pool.view(torch.uint8).long()] * scales.double()[..., None]


def _power(e):
    """2^e of whole numbers, exact on every device (their power function is not)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantise(x):
    """(bytes, scales) of rows x [..., dim] (f32): the least power of two s with |x| <= 448
    s, at least 2^-126, 0 for zeros, NaN for rows that are not finite; then the nearest
    e4m3 value of x / s, ties to even."""
    x = x.double()
    top = x.abs().amax(-1)
    sound = torch.isfinite(top)
    part, power = torch.frexp(torch.where((top > 0) & sound, top, 1.0))  # 1/2 <= part < 1
    s = _power((power - 9 + (part > 0.875).int()).clamp_min(-126))       # 448 = 7/8 2^9
    y = x / s[..., None]
    step = _power(torch.frexp(y.abs().clamp_min(2.0 ** -6))[1] - 4)
    y = torch.where(sound[..., None], torch.round(y / step) * step, 0.0)
    table = e4m3_values()[:127].to(x.device)
    at = torch.searchsorted(table, y.abs().contiguous()).clamp_max(126)
    assert torch.equal(table[at], y.abs())
    bits = (at + torch.where(torch.signbit(y), 128, 0)).to(torch.uint8)
    scales = torch.where(top == 0, 0.0, s)
    return bits, torch.where(sound, scales, float("nan")).float()


def turn_f32(x, cos, sin):
    """x [tokens, heads, dim] rotated in f32, each operation rounded by itself."""
    a, b, c, s = x[..., 0::2].float(), x[..., 1::2].float(), cos[:, None], sin[:, None]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def probabilities(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(distribution, distance of the nucleus' border from a token's, relative) of one row
    of logits, float64."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    out = np.zeros_like(x)
    if not (x > -np.inf).any():
        return out, 1.0
    order = np.lexsort((np.arange(x.size), -x))
    if not temperature > 2.0 ** -100:
        out[order[0]] = 1.0
        return out, 1.0
    top, margin = x[order[0]], 1.0
    if top == np.inf:
        w = (x[order] == np.inf).astype(np.float64)
    elif np.isinf(temperature):
        w = (x[order] > -np.inf).astype(np.float64)
    else:
        w = np.exp((x[order] - top) / temperature)
    if top_k > 0:
        w[top_k:] = 0.0
    if top_p < 1.0:
        before = np.cumsum(w) - w
        some = w[1:] > 0
        if some.any():
            margin = np.abs(before[1:][some] / w.sum() - top_p).min()
        drop = before >= top_p * w.sum()
        drop[0] = False
        w[drop] = 0.0
    if min_p > 0.0 and top < np.inf:
        w[w < min(min_p, 1.0)] = 0.0
    out[order] = w / w.sum()
    return out, margin


def verify(rows, target, draft, drafts, accept, draw):
    """(ids, accepted, margin) of one request of `rows` rows: float64 arrays, draft None
    for proposals made without chance."""
    clean = lambda p: np.where(p > 0, np.minimum(p, 1.0), 0.0)
    ids, margin = [-1] * rows, 1.0
    vocab = target.shape[1]
    stop, q = rows - 1, None
    for r in range(rows - 1):
        x = int(drafts[r])
        p_row = clean(target[r])
        if 0 <= x < vocab:
            q_row = np.eye(1, vocab, x)[0] if draft is None else clean(draft[r])
            if accept[r] * q_row[x] < p_row[x]:
                ids[r] = x
                continue
            q = q_row
        stop = r
        break
    p = clean(target[stop])
    w = p if q is None else np.maximum(p - q, 0.0)
    if not w.sum() > 0:
        w = p
    if w.sum() > 0:
        run = np.cumsum(w)
        u = 0.0 if not draw > 0 else draw
        i = int(np.searchsorted(run, u * run[-1], side="right"))
        if i >= vocab:
            i = int(np.nonzero(w)[0][-1])
        ids[stop] = i if w[i] > 0 else i + int(np.nonzero(w[i:])[0][0])
        if u < 1.0:
            margin = np.abs(run - u * run[-1]).min() / run[-1]
    return ids, stop, margin
