"""Cases of the 8-bit paged cache (appending with the keys' rotation, attention of
new tokens over it) and of speculative decoding (the distribution that sampling
draws from, verification of drafted tokens).

`run` computes a case in plain torch operations, or, with `own` set, by the
package's own entry points.  A cached row is e4m3 elements times one scale, the
least power of two that keeps its largest element within 448."""
import math

import torch

own = False

_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # one new token of one request: the smallest call of a decoding loop (the medium LM's heads)
        dict(name="append8 one token", op="append8", batch=1, new=1, kv=257, heads=16, dim=64, page=16, dtype="f32"),
        # prompts of several requests, ragged, pages that are no power of two
        dict(name="append8 prompts", op="append8", batch=11, new=2048, kv=2500, heads=8, dim=128, page=24, dtype="bf16"),
        # single token, single request, short cache: latency (the medium LM's heads)
        dict(name="attend8 one token", op="attend8", batch=1, new=1, kv=300, qheads=16, heads=16, dim=64, page=16, dtype="f32"),
        # a decoding step of many ragged requests with grouped heads
        dict(name="attend8 decode 64", op="attend8", batch=64, new=1, kv=8192, qheads=32, heads=8, dim=128, page=16, dtype="bf16"),
        # few requests with long caches: the work has to be split along the keys
        dict(name="attend8 long cache", op="attend8", batch=3, new=1, kv=65000, qheads=16, heads=2, dim=128, page=64, dtype="f16"),
        # a step of speculative decoding: four drafted tokens behind the last one of each request
        dict(name="attend8 drafts", op="attend8", batch=32, new=5, kv=4000, qheads=32, heads=8, dim=128, page=16, dtype="bf16"),
        # a chunk of a long prompt over what is cached of it
        dict(name="attend8 chunk", op="attend8", batch=1, new=4096, kv=12000, qheads=32, heads=8, dim=128, page=64, dtype="bf16"),
        # prompts at the trained precision (the medium LM's heads), ragged
        dict(name="attend8 prompts f32", op="attend8", batch=4, new=1024, kv=1024, qheads=16, heads=16, dim=64, page=32, dtype="f32"),
        # one position of one request (the medium LM's vocabulary), filtered
        dict(name="probabilities one row", op="probabilities", rows=1, vocab=32768, dtype="f32", top_k=50, min_p=0.02),
        # the positions of 64 requests with four drafted tokens each
        dict(name="probabilities 320", op="probabilities", rows=320, vocab=128259, dtype="bf16", top_k=40, min_p=0.0),
        # one request (the medium LM's vocabulary)
        dict(name="verify one request", op="verify", batch=1, drafts=4, vocab=32768),
        # a step of many requests
        dict(name="verify 64", op="verify", batch=64, drafts=4, vocab=128259),
    ]


def _log_int(rng, low, high):
    return min(high, int(low * (high / low) ** rng.random() + rng.random()))


def draw(rng):
    op = rng.choice(["append8", "attend8", "attend8", "attend8", "probabilities", "verify"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "probabilities":
        vocab = rng.choice([_log_int(rng, 1000, 128259), 32768, 50257, 128259])
        # 8-bit and speculative decoding rarely run without a filter; no nucleus here: which side of
        # its border a token falls on hangs on the last bits of a sum
        return dict(op=op, rows=min(_log_int(rng, 1, 512), (320 * 128259) // vocab), vocab=vocab, dtype=dtype,
                    top_k=rng.choice([0, 1, 20, 50, 1000]), min_p=rng.choice([0.0, 0.0, 0.05, 0.2]))
    if op == "verify":
        vocab = rng.choice([_log_int(rng, 1000, 128259), 32768, 50257, 128259])
        drafts = rng.choice([1, 2, 4, 4, 7, 11])
        return dict(op=op, batch=max(1, min(_log_int(rng, 1, 256), (320 * 128259) // (vocab * (drafts + 1)))),
                    drafts=drafts, vocab=vocab)
    dim = rng.choice([32, 64, 64, 80, 128, 128, 256])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    if op == "append8":
        batch = _log_int(rng, 1, 256)
        new = rng.choice([1, _log_int(rng, 1, 4096)])
        new = max(1, min(new, 16000 // batch))
        heads = rng.choice([1, 2, 4, 8, 16])
        kv = new + _log_int(rng, 1, 2048)
        kv = max(new, min(kv, 2_000_000_000 // (batch * heads * dim * 8)))
        return dict(op=op, batch=batch, new=new, kv=kv, heads=heads, dim=dim, page=page, dtype=dtype)
    heads = rng.choice([1, 2, 4, 8, 16])
    qheads = heads * rng.choice([1, 2, 4, 8] if heads <= 4 else [1, 2, 4])
    new = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 2, 4096)])
    batch = _log_int(rng, 1, 128)
    batch = max(1, min(batch, 6000 // new))
    kv = new + _log_int(rng, 16, 65000)
    kv = max(new, min(kv, 2_500_000_000 // (batch * heads * dim * 8), 1_200_000_000 // (batch * qheads * new)))
    return dict(op=op, batch=batch, new=new, kv=kv, qheads=qheads, heads=heads, dim=dim, page=page, dtype=dtype)


def _spread(count, low, high):
    """`count` whole numbers between low and high, spread without a pattern; the last is high."""
    return [high if i == count - 1 else low + int((high - low) * ((i * 0.6180339887498949 + 0.37) % 1.0)) for i in range(count)]


def _ragged(case):
    """New tokens and lengths (with them) of each request: a quarter to all of the case's largest."""
    new = _spread(case["batch"], -(-case["new"] // 4), case["new"])
    length = [max(n, m) for n, m in zip(new, _spread(case["batch"], -(-case["kv"] // 4), case["kv"]))]
    return new, length


def _rows_of(case):
    """Rows of each request of a verification: its drafted tokens (some requests have fewer) and one more."""
    return [1 + d for d in _spread(case["batch"], case["drafts"] // 2, case["drafts"])]


def _rope_tables(length, dim, device):
    inv = (10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)).float()
    angle = (torch.arange(length, dtype=torch.float32, device=device)[:, None] * inv[None, :]).double()
    return angle.cos().float(), angle.sin().float()


def _quantise(x):
    """e4m3 elements and scale of f32 rows: x / s, s the least power of two with |x| <= 448 s; 0 for rows of zeros."""
    top = x.abs().amax(-1)
    part, power = torch.frexp(top)  # top = part 2^power, 1/2 <= part < 1; 448 = 7/8 2^9
    scale = torch.ldexp(torch.ones_like(top), power - 9 + (part > 0.875).int())
    scale = torch.where(top > 0, scale, 0.0)
    return (x / torch.where(top > 0, scale, 1.0)[..., None]).to(_E4M3), scale


def _probabilities(logits, temperature):
    return torch.softmax(logits / temperature, -1)


def _language_logits(normal, g, rows, vocab):
    # logits of a language model: a broad bulk, a handful of likely tokens, an end of the
    # vocabulary that is never allowed
    logits = normal(rows, vocab) * 2.0
    at = torch.randint(vocab, (rows, 24), device="cuda", generator=g)
    logits.scatter_add_(1, at, 9.0 - 0.3 * torch.arange(24, device="cuda", dtype=torch.float32).expand(rows, 24))
    logits[:, vocab - vocab // 200:] = -math.inf
    return logits


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "probabilities":
        rows, vocab = case["rows"], case["vocab"]
        logits = _language_logits(normal, g, rows, vocab)
        # one row in eight decodes greedily; the others are spread around temperature 0.9
        temperature = 0.6 + 0.6 * torch.rand(rows, device="cuda", generator=g)
        temperature[7::8] = 0.0
        return dict(case=case, logits=logits.to(_DTYPE[case["dtype"]]), temperature=temperature,
                    top_k=torch.full((rows,), case["top_k"], device="cuda", dtype=torch.int64),
                    min_p=torch.full((rows,), case["min_p"], device="cuda"),
                    probs=torch.zeros(rows, vocab, device="cuda"))
    if case["op"] == "verify":
        rows, vocab = _rows_of(case), case["vocab"]
        tokens = sum(rows)
        logits = _language_logits(normal, g, tokens, vocab)
        # a draft model that mostly agrees: its logits are the target's with some noise
        target = _probabilities(logits, 0.8)
        draft = _probabilities(logits + 0.5 * normal(tokens, vocab), 0.8)
        u = torch.rand(tokens, 1, device="cuda", generator=g, dtype=torch.float64)
        run_sum = draft.double().cumsum(1)
        drafts = torch.searchsorted(run_sum, u * run_sum[:, -1:], right=True)[:, 0].clamp_max(vocab - 1)
        offsets = [0]
        for n in rows:
            offsets.append(offsets[-1] + n)
        return dict(case=case, target=target, draft=draft, drafts=drafts, tokens=tokens,
                    offsets=torch.tensor(offsets, device="cuda"),
                    accept=torch.rand(tokens, device="cuda", generator=g),
                    uniform=torch.rand(case["batch"], device="cuda", generator=g),
                    ids=torch.zeros(tokens, device="cuda", dtype=torch.int64),
                    accepted=torch.zeros(case["batch"], device="cuda", dtype=torch.int64))
    t = _DTYPE[case["dtype"]]
    batch, heads, dim, page = case["batch"], case["heads"], case["dim"], case["page"]
    new, length = _ragged(case)
    columns = -(-case["kv"] // page)
    pages = batch * columns + 3  # more than are used
    table = torch.randperm(pages, device="cuda", generator=g)[:batch * columns].reshape(batch, columns).int()
    cos, sin = _rope_tables(case["kv"], dim, "cuda")
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    # cached rows whose sizes differ, as those of a model's tokens do
    keys, key_scales = _quantise(normal(pages, heads, page, dim) * (0.5 * normal(pages, heads, page, 1)).exp())
    values, value_scales = _quantise(normal(pages, heads, page, dim) * (0.5 * normal(pages, heads, page, 1)).exp())
    s = dict(case=case, keys=keys, values=values, key_scales=key_scales, value_scales=value_scales,
             table=table, cos=cos, sin=sin, offsets=torch.tensor(offsets, device="cuda"),
             lengths=torch.tensor(length, device="cuda"), tokens=offsets[-1])
    if case["op"] == "append8":
        # the key and value parts of a fused projection's output
        both = normal(s["tokens"], 2, heads, dim).to(t)
        s["k"], s["v"] = both[:, 0], both[:, 1]
    else:
        s["q"] = normal(s["tokens"], case["qheads"], dim).to(t)
        s["o"] = torch.zeros_like(s["q"])
    return s


def _places(s):
    """Request and position of every new token."""
    token = torch.arange(s["tokens"], device="cuda")
    request = torch.searchsorted(s["offsets"], token, right=True) - 1
    return request, token - s["offsets"][request + 1] + s["lengths"][request]


def _rotated(x, cos, sin):
    """x [tokens, heads, dim] in 32 bits, pairs (2i, 2i + 1) turned by the angles of cos, sin [tokens, dim / 2]."""
    a, b = x[..., 0::2].float(), x[..., 1::2].float()
    c, s = cos[:, None], sin[:, None]
    return torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)


def _cache(s):
    return {n: s[n] for n in ("keys", "values", "key_scales", "value_scales")}


def _plain_append8(s):
    page = s["case"]["page"]
    request, at = _places(s)
    where = s["table"][request, at // page].long()
    for name, x in (("key", _rotated(s["k"], s["cos"][at], s["sin"][at])), ("value", s["v"].float())):
        bits, scale = _quantise(x)
        s[name + "s"].view(torch.uint8)[where, :, at % page] = bits.view(torch.uint8)
        s[name + "_scales"][where, :, at % page] = scale
    return _cache(s)


def _plain_attend8(s):
    case = s["case"]
    batch, new, kv, heads, dim = case["batch"], case["new"], case["kv"], case["heads"], case["dim"]
    group, table = case["qheads"] // heads, s["table"].long()
    request, at = _places(s)
    index = torch.arange(s["tokens"], device="cuda") - s["offsets"][request]
    # queries padded to the longest chunk: [batch, heads, group * new, dim]
    q = torch.zeros(batch, new, heads, group, dim, device="cuda")
    q[request, index] = _rotated(s["q"], s["cos"][at], s["sin"][at]).unflatten(1, (heads, group))
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)

    def rows(bits, scales):
        x = bits.view(torch.uint8)[table].permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :kv].view(_E4M3).float()
        return x.mul_(scales[table].permute(0, 2, 1, 3).flatten(2)[:, :, :kv, None])

    k, v = rows(s["keys"], s["key_scales"]), rows(s["values"], s["value_scales"])
    score = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(dim))
    position = torch.full((batch, new), -1, device="cuda")
    position[request, index] = at
    seen = torch.arange(kv, device="cuda") <= position[:, :, None]
    score = score.unflatten(2, (group, new)).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-1e30)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    o = torch.matmul(weight.flatten(2, 3), v).unflatten(2, (group, new)) / total
    o = o.permute(0, 3, 1, 2, 4)[request, index]
    return {"o": o.flatten(1, 2).to(s["q"].dtype)}


def _plain_probabilities(s):
    x = s["logits"].double()  # borders between tokens need more than 32 bits
    rows, vocab = x.shape
    x, token = torch.sort(x, dim=1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    weight = ((x - x[:, :1]) / torch.where(t > 0, t, 1.0)).exp()
    rank = torch.arange(vocab, device="cuda")
    top_k = torch.where(t > 0, s["top_k"][:, None], 1)
    keep = ((rank < top_k) | (top_k <= 0)) & (weight >= s["min_p"].double()[:, None])
    weight = weight * keep
    return {"probs": torch.zeros_like(weight).scatter_(1, token, weight / weight.sum(1, keepdim=True)).float()}


def _plain_verify(s):
    offsets, drafts, tokens = s["offsets"], s["drafts"], s["tokens"]
    token = torch.arange(tokens, device="cuda")
    request = torch.searchsorted(offsets, token, right=True) - 1
    last = token == offsets[request + 1] - 1
    p = s["target"].gather(1, drafts[:, None])[:, 0].double()
    q = s["draft"].gather(1, drafts[:, None])[:, 0].double()
    good = (s["accept"].double() * q < p) & ~last
    # the first row of each request that is not accepted: its drafted tokens end there
    stop = torch.full((s["case"]["batch"],), tokens, device="cuda").scatter_reduce_(
        0, request, torch.where(good, tokens, token), "amin")
    accepted = stop - offsets[:-1]
    row = s["target"][stop].double()
    rest = (row - s["draft"][stop].double()).clamp_min(0.0)
    rest = torch.where((last[stop] | (rest.sum(1) <= 0.0))[:, None], row, rest)
    run_sum = rest.cumsum(1)
    drawn = (run_sum > s["uniform"].double()[:, None] * run_sum[:, -1:]).int().argmax(1)
    ids = torch.where(token < stop[request], drafts, torch.where(token == stop[request], drawn[request], -1))
    return {"ids": ids, "accepted": accepted}


def _paged8(s):
    from eshkol_transformer_b200 import paged
    cache = paged.PagedCache8(s["keys"], s["values"], s["key_scales"], s["value_scales"], _DTYPE[s["case"]["dtype"]])
    batch = paged.PagedBatch(s["offsets"], s["lengths"], s["table"], s["tokens"], s["case"]["new"], s["case"]["kv"])
    return paged, cache, batch


def _own_append8(s):
    if "cache" not in s:  # what a serving loop keeps
        _, s["cache"], s["batch"] = _paged8(s)
    s["cache"].append(s["batch"], s["k"], s["v"], rope=(s["cos"], s["sin"]))
    return _cache(s)


def _own_attend8(s):
    if "attention" not in s:
        paged, cache, s["batch"] = _paged8(s)
        s["attention"] = paged.PagedAttention(cache, s["case"]["qheads"])
    s["attention"].forward(s["batch"], s["q"], s["o"], rope=(s["cos"], s["sin"]))
    return {"o": s["o"]}


def _own_probabilities(s):
    from eshkol_transformer_b200 import sampling
    if "sampler" not in s:
        s["sampler"] = sampling.Sampler(s["case"]["rows"], s["case"]["vocab"])
    s["sampler"].probabilities(s["logits"], s["probs"], temperature=s["temperature"], top_k=s["top_k"], min_p=s["min_p"])
    return {"probs": s["probs"]}


def _own_verify(s):
    from eshkol_transformer_b200 import sampling
    if "verifier" not in s:
        s["verifier"] = sampling.Verifier(s["case"]["batch"], s["tokens"], s["case"]["vocab"])
    s["verifier"].verify(s["offsets"], s["target"], s["drafts"], s["draft"], s["accept"], s["uniform"], s["ids"], s["accepted"])
    return {"ids": s["ids"], "accepted": s["accepted"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append8": _own_append8, "attend8": _own_attend8, "probabilities": _own_probabilities, "verify": _own_verify}[op](state)
    return {"append8": _plain_append8, "attend8": _plain_attend8, "probabilities": _plain_probabilities, "verify": _plain_verify}[op](state)


def work(case):
    if case["op"] == "probabilities":
        n = case["rows"] * case["vocab"]
        # per logit: a difference, a product, an exponential, a comparison, a sum, a product
        return {"bytes": n * (_SIZE[case["dtype"]] + 4) + case["rows"] * (4 + 8 + 4), "flops": 6 * n}
    if case["op"] == "verify":
        rows = _rows_of(case)
        # two rows of probabilities per request, two values per drafted token
        return {"bytes": case["batch"] * (2 * 4 * case["vocab"] + 4 + 8 + 8) + 8 + sum(rows) * (8 + 4 + 2 * 4 + 8),
                "flops": 3 * case["batch"] * case["vocab"]}
    size = _SIZE[case["dtype"]]
    new, length = _ragged(case)
    tokens, wide = sum(new), case["heads"] * case["dim"]
    cached = case["heads"] * (case["dim"] + 4)  # bytes of a token's keys, and of its values
    meta = 16 * case["batch"] + 8 + 4 * sum(-(-m // case["page"]) for m in length)
    tables = min(4 * case["dim"] * max(length), 4 * case["dim"] * tokens)
    if case["op"] == "append8":
        return {"bytes": 2 * tokens * (wide * size + cached) + tables + meta, "flops": 7 * tokens * wide}
    seen = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, length))
    qwide = case["qheads"] * case["dim"]
    return {"bytes": 2 * sum(length) * cached + 2 * tokens * qwide * size + tables + meta, "flops": 4 * seen * qwide}


def _exact_turn(x, angle_cos, angle_sin):
    z = torch.view_as_complex(x.double().unflatten(-1, (-1, 2)).contiguous())
    return torch.view_as_real(z * torch.complex(angle_cos.double(), angle_sin.double())[:, None]).flatten(-2)


def _exact_value(bits):
    """What bytes of type e4m3 stand for: sign, 4 bits of exponent (bias 7), 3 of fraction; exponent 0: multiples of 2^-9."""
    b = torch.arange(256, dtype=torch.float64, device=bits.device)
    low = b % 128
    e, f = torch.floor(low / 8), low % 8
    table = torch.where(e > 0, (1 + f / 8) * 2.0 ** (e - 7), f * 2.0 ** -9) * torch.where(b >= 128, -1.0, 1.0)
    return table[bits.view(torch.uint8).int()]


def _exact_round(y):
    """y (|y| <= 448) to the nearest of type e4m3, ties to even."""
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "probabilities":
        return _exact_probabilities(s)
    if case["op"] == "verify":
        return None  # whole numbers only
    page = case["page"]
    new, length = _ragged(case)
    if case["op"] == "append8":
        out = {"keys": _exact_value(s["keys"]), "values": _exact_value(s["values"]),
               "key_scales": s["key_scales"].double(), "value_scales": s["value_scales"].double()}
    else:
        out = {"o": torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")}
    first = 0
    for b, (n, m) in enumerate(zip(new, length)):
        rows = slice(first, first + n)
        first += n
        chain = s["table"][b].long()
        cos, sin = s["cos"][m - n:m], s["sin"][m - n:m]
        if case["op"] == "append8":
            slot = torch.arange(m - n, m, device="cuda")
            for name, x in (("key", _exact_turn(s["k"][rows], cos, sin)), ("value", s["v"][rows].double())):
                scale = 2.0 ** torch.ceil(torch.log2(x.abs().amax(-1) / 448.0))
                out[name + "_scales"][chain[slot // page], :, slot % page] = scale
                out[name + "s"][chain[slot // page], :, slot % page] = _exact_round(x / scale[..., None])
            continue
        q = _exact_turn(s["q"][rows], cos, sin)
        group = case["qheads"] // case["heads"]
        hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
        for h in range(case["heads"]):
            k, v = ((_exact_value(x[chain, h]) * y[chain, h].double()[..., None]).flatten(0, 1)[:m]
                    for x, y in ((s["keys"], s["key_scales"]), (s["values"], s["value_scales"])))
            for j in range(h * group, (h + 1) * group):
                a = (q[:, j] @ k.T / math.sqrt(case["dim"])).masked_fill_(hidden, -math.inf)
                out["o"][rows, j] = torch.softmax(a, 1) @ v
    return out


def _exact_probabilities(s):
    probs = torch.zeros(s["logits"].shape, dtype=torch.float64, device="cuda")
    for r in range(s["case"]["rows"]):
        x, t = s["logits"][r].double(), float(s["temperature"][r])
        order = torch.argsort(x, descending=True, stable=True)
        if t == 0.0:
            probs[r, order[0]] = 1.0
            continue
        w = torch.softmax(x[order] / t, 0)
        k, low = int(s["top_k"][r]), float(s["min_p"][r])
        if k > 0:
            w[k:] = 0.0
        w[w < low * w[0]] = 0.0
        probs[r, order] = w / w.sum()
    return {"probs": probs}
