"""Cases of the serving operators: appending keys and values to a paged cache
(with the keys' position rotation), attention of new tokens over that cache,
and sampling the next token from logits.

`run` computes a case in plain torch operations, or, with `own` set, by the
package's own entry points."""
import math

import torch

own = False

_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one new token of one request: the smallest call of a decoding loop (the medium LM's heads)
        dict(name="append one token", op="append", batch=1, new=1, kv=257, heads=16, dim=64, page=16, dtype="f32"),
        # a decoding step of many requests
        dict(name="append decode 256", op="append", batch=256, new=1, kv=2000, heads=8, dim=128, page=16, dtype="bf16"),
        # prompts of several requests, ragged, pages that are no power of two
        dict(name="append prompts", op="append", batch=11, new=2048, kv=2500, heads=8, dim=128, page=24, dtype="f16"),
        # single token, single request, short cache: latency (the medium LM's heads)
        dict(name="attend one token", op="attend", batch=1, new=1, kv=300, qheads=16, heads=16, dim=64, page=16, dtype="f32"),
        # a decoding step of many ragged requests with grouped heads
        dict(name="attend decode 64", op="attend", batch=64, new=1, kv=8192, qheads=32, heads=8, dim=128, page=16, dtype="bf16"),
        # few requests with long caches: the work has to be split along the keys
        dict(name="attend long cache", op="attend", batch=3, new=1, kv=65000, qheads=16, heads=2, dim=128, page=64, dtype="f16"),
        # a chunk of a long prompt over what is cached of it
        dict(name="attend chunk", op="attend", batch=1, new=4096, kv=12000, qheads=32, heads=8, dim=128, page=64, dtype="bf16"),
        # prompts at the trained precision (the medium LM's heads), ragged
        dict(name="attend prompts f32", op="attend", batch=4, new=1024, kv=1100, qheads=16, heads=16, dim=64, page=16, dtype="f32"),
        # one row with every filter on (the medium LM's vocabulary)
        dict(name="sample one row", op="sample", rows=1, vocab=32768, dtype="f32", top_k=50, top_p=0.9, min_p=0.02),
        # a decoding step's rows, nucleus only
        dict(name="sample nucleus", op="sample", rows=64, vocab=32768, dtype="f32", top_k=0, top_p=0.95, min_p=0.0),
        # many rows, a large odd vocabulary, top-k and top-p
        dict(name="sample 256 wide", op="sample", rows=256, vocab=128259, dtype="bf16", top_k=40, top_p=0.95, min_p=0.0),
        # no filter but the temperature: the whole distribution is kept
        dict(name="sample whole", op="sample", rows=128, vocab=50257, dtype="f32", top_k=0, top_p=1.0, min_p=0.0),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sample"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "sample":
        vocab = _log_int(rng, 1000, 131072)
        return dict(op=op, rows=min(_log_int(rng, 1, 512), (256 * 128259) // vocab), vocab=vocab, dtype=dtype,
                    top_k=rng.choice([0, 1, 20, 50, 1000]), top_p=rng.choice([0.3, 0.8, 0.95, 1.0]),
                    min_p=rng.choice([0.0, 0.0, 0.05, 0.2]))
    dim = rng.choice([32, 64, 64, 80, 128, 128, 256])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    if op == "append":
        batch = _log_int(rng, 1, 256)
        new = rng.choice([1, _log_int(rng, 1, 4096)])
        new = max(1, min(new, 16000 // batch))
        heads = rng.choice([1, 2, 4, 8, 16])
        kv = new + _log_int(rng, 1, 2048)
        kv = max(new, min(kv, 2_000_000_000 // (batch * heads * dim * 8)))
        return dict(op=op, batch=batch, new=new, kv=kv, heads=heads, dim=dim, page=page, dtype=dtype)
    heads = rng.choice([1, 2, 4, 8, 16])
    qheads = heads * rng.choice([1, 2, 4, 8] if heads <= 4 else [1, 2, 4])
    new = rng.choice([1, 1, _log_int(rng, 2, 4096)])
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


def _rope_tables(length, dim, device):
    inv = (10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)).float()
    angle = (torch.arange(length, dtype=torch.float32, device=device)[:, None] * inv[None, :]).double()
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # logits of a language model: a broad bulk, a handful of likely tokens, an end of the
        # vocabulary that is never allowed
        logits = normal(rows, vocab) * 2.0
        at = torch.randint(vocab, (rows, 24), device="cuda", generator=g)
        logits.scatter_add_(1, at, 9.0 - 0.3 * torch.arange(24, device="cuda", dtype=torch.float32).expand(rows, 24))
        logits[:, vocab - vocab // 200:] = -math.inf
        u = torch.rand(rows, device="cuda", generator=g)
        # one row in eight decodes greedily; the others are spread around temperature 0.9
        temperature = 0.6 + 0.6 * torch.rand(rows, device="cuda", generator=g)
        temperature[7::8] = 0.0
        return dict(case=case, logits=logits.to(_DTYPE[case["dtype"]]), u=u, temperature=temperature,
                    top_k=torch.full((rows,), case["top_k"], device="cuda", dtype=torch.int64),
                    top_p=torch.full((rows,), case["top_p"], device="cuda"),
                    min_p=torch.full((rows,), case["min_p"], device="cuda"),
                    ids=torch.zeros(rows, device="cuda", dtype=torch.int64),
                    logprobs=torch.zeros(rows, device="cuda"))
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
    s = dict(case=case, keys=normal(pages, heads, page, dim).to(t), values=normal(pages, heads, page, dim).to(t),
             table=table, cos=cos, sin=sin, offsets=torch.tensor(offsets, device="cuda"),
             lengths=torch.tensor(length, device="cuda"), tokens=offsets[-1])
    if case["op"] == "append":
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


def _plain_append(s):
    page = s["case"]["page"]
    request, at = _places(s)
    where = s["table"][request, at // page].long()
    s["keys"][where, :, at % page] = _rotated(s["k"], s["cos"][at], s["sin"][at]).to(s["k"].dtype)
    s["values"][where, :, at % page] = s["v"]
    return {"keys": s["keys"], "values": s["values"]}


def _plain_attend(s):
    case = s["case"]
    batch, new, kv, heads, dim = case["batch"], case["new"], case["kv"], case["heads"], case["dim"]
    group = case["qheads"] // heads
    request, at = _places(s)
    index = torch.arange(s["tokens"], device="cuda") - s["offsets"][request]
    # queries padded to the longest chunk: [batch, heads, group * new, dim]
    q = torch.zeros(batch, new, heads, group, dim, device="cuda")
    q[request, index] = _rotated(s["q"], s["cos"][at], s["sin"][at]).unflatten(1, (heads, group))
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)
    k, v = (p[s["table"].long()].permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :kv].float() for p in (s["keys"], s["values"]))
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


def _plain_sample(s):
    x = s["logits"].double()  # borders between tokens need more than 32 bits
    rows, vocab = x.shape
    x, token = torch.sort(x, dim=1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    weight = ((x - x[:, :1]) / torch.where(t > 0, t, 1.0)).exp()
    rank = torch.arange(vocab, device="cuda")
    top_k = torch.where(t > 0, s["top_k"][:, None], 1)
    keep = (rank < top_k) | (top_k <= 0)
    kept = weight * keep
    before = kept.cumsum(1) - kept
    keep &= (before < s["top_p"].double()[:, None] * kept.sum(1, keepdim=True)) | (s["top_p"] >= 1)[:, None]
    keep &= weight >= s["min_p"].double()[:, None]
    weight = weight * keep
    in_order = torch.zeros_like(weight).scatter_(1, token, weight)
    run_sum = in_order.cumsum(1)
    total = run_sum[:, -1:]
    ids = (run_sum > s["u"].double()[:, None] * total).int().argmax(1)
    logprobs = (in_order.gather(1, ids[:, None]) / total).log()[:, 0].float()
    return {"ids": ids, "logprobs": logprobs}


def _own_append(s):
    from eshkol_transformer_b200 import paged
    if "cache" not in s:  # what a serving loop keeps
        s["cache"] = paged.PagedCache(s["keys"], s["values"])
        s["batch"] = paged.PagedBatch(s["offsets"], s["lengths"], s["table"], s["tokens"], s["case"]["new"], s["case"]["kv"])
    s["cache"].append(s["batch"], s["k"], s["v"], rope=(s["cos"], s["sin"]))
    return {"keys": s["keys"], "values": s["values"]}


def _own_attend(s):
    from eshkol_transformer_b200 import paged
    if "attention" not in s:
        s["attention"] = paged.PagedAttention(paged.PagedCache(s["keys"], s["values"]), s["case"]["qheads"])
        s["batch"] = paged.PagedBatch(s["offsets"], s["lengths"], s["table"], s["tokens"], s["case"]["new"], s["case"]["kv"])
    s["attention"].forward(s["batch"], s["q"], s["o"], rope=(s["cos"], s["sin"]))
    return {"o": s["o"]}


def _own_sample(s):
    from eshkol_transformer_b200 import sampling
    if "sampler" not in s:
        s["sampler"] = sampling.Sampler(s["case"]["rows"], s["case"]["vocab"])
    s["sampler"].sample(s["logits"], s["u"], s["ids"], s["logprobs"], temperature=s["temperature"], top_k=s["top_k"],
                        top_p=s["top_p"], min_p=s["min_p"])
    return {"ids": s["ids"], "logprobs": s["logprobs"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "sample": _own_sample}[op](state)
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[op](state)


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        # per logit: a difference, a product, an exponential, a comparison, a sum
        return {"bytes": n * size + case["rows"] * (4 * 4 + 8 + 8 + 4), "flops": 5 * n}
    new, length = _ragged(case)
    tokens, row = sum(new), case["heads"] * case["dim"] * size
    meta = 16 * case["batch"] + 8 + 4 * sum(-(-m // case["page"]) for m in length)
    tables = 4 * case["dim"] * max(length)
    if case["op"] == "append":
        return {"bytes": 4 * tokens * row + min(tables, 4 * case["dim"] * tokens) + meta, "flops": 3 * tokens * case["heads"] * case["dim"]}
    seen = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, length))
    wide = case["qheads"] * case["dim"]
    return {"bytes": 2 * sum(length) * row + 2 * tokens * wide * size + min(tables, 4 * case["dim"] * tokens) + meta,
            "flops": 4 * seen * wide}


def _exact_turn(x, angle_cos, angle_sin):
    z = torch.view_as_complex(x.double().unflatten(-1, (-1, 2)).contiguous())
    return torch.view_as_real(z * torch.complex(angle_cos.double(), angle_sin.double())[:, None]).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    page, out = case["page"], {}
    new, length = _ragged(case)
    if case["op"] == "append":
        out = {"keys": s["keys"].double(), "values": s["values"].double()}
    else:
        out = {"o": torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")}
    first = 0
    for b, (n, m) in enumerate(zip(new, length)):
        rows = slice(first, first + n)
        first += n
        chain = s["table"][b].long()
        cos, sin = s["cos"][m - n:m], s["sin"][m - n:m]
        if case["op"] == "append":
            slot = torch.arange(m - n, m, device="cuda")
            flat = chain[slot // page] * page + slot % page
            for name, x in (("keys", _exact_turn(s["k"][rows], cos, sin)), ("values", s["v"][rows].double())):
                pool = out[name].transpose(1, 2).flatten(0, 1)
                pool[flat] = x
                out[name] = pool.unflatten(0, (-1, page)).transpose(1, 2).contiguous()
            continue
        q = _exact_turn(s["q"][rows], cos, sin)
        group = case["qheads"] // case["heads"]
        hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
        for h in range(case["heads"]):
            k, v = (p[chain, h].flatten(0, 1)[:m].double() for p in (s["keys"], s["values"]))
            for j in range(h * group, (h + 1) * group):
                a = (q[:, j] @ k.T / math.sqrt(case["dim"])).masked_fill_(hidden, -math.inf)
                out["o"][rows, j] = torch.softmax(a, 1) @ v
    return out


def _exact_sample(s):
    logprobs = []
    for r in range(s["case"]["rows"]):
        x, t = s["logits"][r].double(), float(s["temperature"][r])
        if t == 0.0:
            logprobs.append(0.0)
            continue
        order = torch.argsort(x, descending=True, stable=True)
        w = torch.softmax(x[order] / t, 0)
        k, p, low = int(s["top_k"][r]), float(s["top_p"][r]), float(s["min_p"][r])
        if k > 0:
            w[k:] = 0.0
        if p < 1.0:
            mass = w / w.sum()
            w[mass.cumsum(0) - mass >= p] = 0.0
        w[w < low * w[0]] = 0.0
        at = torch.zeros_like(w)
        at[order] = w
        c = at.cumsum(0)
        i = int(torch.searchsorted(c, c[-1] * float(s["u"][r]), right=True))
        logprobs.append(math.log(float(at[i] / c[-1])))
    return {"ids": None, "logprobs": torch.tensor(logprobs, dtype=torch.float64, device="cuda")}
