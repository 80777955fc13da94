"""Speculative decoding's operators: the distributions that sampling draws from and the
verification of drafted tokens, against plain float64 forms, alone and in a loop with the
8-bit cache.

Tolerances.  A weight is an f32 whose exponent is formed in two steps, off by at most
2^-22.5 (1.7e-7) of itself (1e-7 and its rounding), the total (integers of 2^-35) by 1e-7
and, for n tokens, n 2^-36 of the largest weight, which is at most the total; the product
with the reciprocal by two roundings: 4e-7 + n 2^-36 of a probability, and tokens below
2^-36 of the likeliest may be 0.  Verification compares whole numbers, wherever a draw is
not within 1e-6 of a border: its weights are f32 differences (2^-24 of each), its sums
float64.
"""
import math

import numpy as np
import pytest
import torch

from cache8_f64 import probabilities, quantise, rows_of, turn_f32, verify
from eshkol_transformer_b200 import paged, sampling
from serving_f64 import attention, rope_tables, turn

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def logits_of(rows, vocab, dtype, seed, sigma=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, vocab, device="cuda", generator=g) * sigma
    if vocab > 50:
        x[:, vocab - vocab // 50:] = -math.inf
        x[:, :24] += 9.0 - 0.3 * torch.arange(24, device="cuda")
        x = x[:, torch.randperm(vocab, device="cuda", generator=g)].contiguous()
    return x.to(dtype)


def filters(rows, temperature=None, top_k=None, top_p=None, min_p=None):
    dev = lambda a, t: None if a is None else torch.as_tensor(np.broadcast_to(a, rows).copy(), dtype=t, device="cuda")
    return dict(temperature=dev(temperature, F32), top_k=dev(top_k, torch.int64), top_p=dev(top_p, F32),
                min_p=dev(min_p, F32))


def distributions(x, out=None, **kw):
    out = torch.full(x.shape, 7.0, device="cuda") if out is None else out
    sampling.Sampler(*x.shape).probabilities(x, out, **filters(x.shape[0], **kw))
    return out


def check_distributions(x, temperature=None, top_k=None, top_p=None, min_p=None, least=0.5):
    got = distributions(x, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p).cpu().numpy()
    xs, (rows, vocab) = x.double().cpu().numpy(), x.shape
    at = lambda a, r, off: off if a is None else float(np.float32(np.broadcast_to(a, rows)[r]))
    checked = 0
    for r in range(rows):
        want, margin = probabilities(xs[r], at(temperature, r, 1.0), int(at(top_k, r, 0)), at(top_p, r, 1.0),
                                     at(min_p, r, 0.0))
        if margin <= 2.5e-7:  # which side of the nucleus' border a token is on
            continue
        checked += 1
        low = want.max() * 2.0 ** -36 * 1.001
        off = np.abs(got[r] - want)
        assert (off <= (4e-7 + vocab * 2.0 ** -36) * want + np.where(want <= low, low, 0.0)).all(), (r, off.max())
        assert (got[r][want == 0] == 0).all()
        assert want.sum() == 0 or abs(got[r].astype(np.float64).sum() - 1) <= 4e-7 + 2 * vocab * 2.0 ** -36
    assert checked >= least * rows


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 4099, 32768, 50257])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05),
                                dict(top_k=50, top_p=0.8, min_p=0.02), dict(top_k=3000), dict(top_k=1),
                                dict(top_p=0.0), dict(min_p=1.0), dict(top_k=700)], ids=str)
def test_distributions_vs_float64(lib, cuda, vocab, dtype, kw):
    t = np.linspace(0.3, 1.7, 12).astype(np.float32)
    t[5] = 0.0
    check_distributions(logits_of(12, vocab, dtype, vocab), t, **kw)


@pytest.mark.parametrize("dtype,vocab", [(F32, 128259), (BF16, 128259), (F32, 300001), (BF16, 450001), (F32, 450001)])
def test_distributions_of_large_vocabularies(lib, cuda, vocab, dtype):
    """Rows over a whole cluster and beyond its shared memory."""
    x = logits_of(3, vocab, dtype, 6, sigma=1.0)
    x[:, 1000:1010] += 14.0
    for kw in (dict(), dict(top_k=64), dict(top_k=5, top_p=0.5), dict(min_p=0.3), dict(top_k=1000),
               dict(temperature=0.0)):
        check_distributions(x, least=0.0 if "top_p" in kw else 1.0, **kw)


def test_distributions_special_values(lib, cuda):
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf, -inf, -inf, -inf], [nan, nan, -inf, nan], [nan, -inf, 3.0, nan], [1.0, inf, -inf, inf],
                      [-3e38, 3e38, 0.0, nan], [0.0, -0.0, -inf, nan], [-65504.0] * 4], device="cuda")
    none, last = [0.0] * 4, [0.0, 0.0, 1.0, 0.0]
    want = [none, none, last, [0, 0.5, 0, 0.5], [0, 1, 0, 0], [0.5, 0.5, 0, 0], [0.25] * 4]
    assert distributions(x).tolist() == want
    assert distributions(x, top_k=2).tolist() == want[:6] + [[0.5, 0.5, 0.0, 0.0]]
    assert distributions(x, temperature=0.0).tolist() == [none, none, last, [0, 1, 0, 0], [0, 1, 0, 0], [1, 0, 0, 0],
                                                          [1, 0, 0, 0]]
    assert distributions(x, temperature=nan)[3].tolist() == [0, 1, 0, 0]
    hot = distributions(x[4:], temperature=inf).tolist()
    assert hot == [[np.float32(1 / 3)] * 3 + [0.0], [0.5, 0.5, 0, 0], [0.25] * 4]
    many = torch.zeros(2, 30011, device="cuda")  # thousands of equal logits: ties by index
    got = distributions(many, top_k=300)
    assert (got[:, :300] == np.float32(1 / 300)).all() and (got[:, 300:] == 0).all()
    got = distributions(many, top_p=0.25)
    kept = math.ceil(30011 / 4)
    assert (got[:, :kept] > 0).all() and (got[:, kept:] == 0).all()


@pytest.mark.parametrize("kw", [dict(), dict(top_k=20), dict(temperature=0.0), dict(top_k=600, top_p=0.9)], ids=str)
def test_distributions_strides(lib, cuda, kw):
    """Logits and probabilities inside larger tensors, at every alignment; nothing beside
    them is written, and every element is."""
    for vocab, off in ((5003, 1), (5003, 2), (5003, 3), (20000, 0)):
        for dtype in (F32, BF16):
            wide = torch.zeros(5, vocab + 9, device="cuda", dtype=dtype)
            x = wide[:, off:off + vocab]
            x.copy_(logits_of(5, vocab, dtype, vocab))
            out = torch.full((5, vocab + 11), 7.0, device="cuda")
            inside = out[:, 3 - off + 1:3 - off + 1 + vocab]
            distributions(x, inside, **kw)
            assert torch.equal(inside, distributions(x.contiguous(), **kw))
            out[:, 3 - off + 1:3 - off + 1 + vocab] = 7.0
            assert (out == 7.0).all()


@pytest.mark.parametrize("kw", [dict(), dict(top_k=20), dict(temperature=0.0)], ids=str)
def test_distributions_beside_their_logits(lib, cuda, kw):
    """Rows of logits and of probabilities that alternate in one tensor share no byte; in place
    they would, and are refused."""
    x = logits_of(5, 1003, F32, 3)
    both = torch.full((5, 2 * 1003), 7.0, device="cuda")
    both[:, :1003] = x
    got = distributions(both[:, :1003], both[:, 1003:], **kw)
    want = distributions(x, **kw)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(both[:, :1003], x)
    for at in (0, 1002):
        with pytest.raises(RuntimeError):
            distributions(both[:, :1003], both[:, at:at + 1003], **kw)


def test_draws_have_their_probability(lib, cuda):
    """What sample draws from the same logits is kept, with this probability."""
    x, rows = logits_of(64, 20000, BF16, 3), 64
    for kw in (dict(), dict(top_k=30), dict(top_p=0.8), dict(top_k=500, top_p=0.9, min_p=0.001)):
        f = filters(rows, temperature=0.8, **kw)
        ids, lp = torch.empty(rows, dtype=torch.int64, device="cuda"), torch.empty(rows, device="cuda")
        s = sampling.Sampler(rows, 20000)
        s.sample(x, torch.rand(rows, device="cuda"), ids, lp, **f)
        p = torch.empty(rows, 20000, device="cuda")
        s.probabilities(x, p, **f)
        at = p.gather(1, ids[:, None])[:, 0]
        assert (at > 0).all() and torch.allclose(at.log(), lp, atol=2e-6)


# ---- verification ---------------------------------------------------------------------------

class Drafts:
    def __init__(self, rows, vocab, seed=1, agree=0.5, filtered=False, spare=2, chance=True):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.rows, self.vocab = rows, vocab
        offsets = np.concatenate([[0], np.cumsum(rows)]).astype(np.int64)
        self.tokens = int(offsets[-1]) + spare
        x = torch.randn(self.tokens, vocab, device="cuda", generator=g) * 2
        noise = torch.randn(self.tokens, vocab, device="cuda", generator=g)
        self.target, self.draft = torch.softmax(x, 1), torch.softmax(x + agree * noise, 1)
        if filtered:
            for p in (self.target, self.draft):
                p *= p >= p.topk(min(vocab, 5), 1)[0][:, -1:]
                p /= p.sum(1, keepdim=True)
        self.drafts = torch.multinomial(self.draft, 1, generator=g)[:, 0]
        self.accept = torch.rand(self.tokens, device="cuda", generator=g)
        self.draw = torch.rand(len(rows), device="cuda", generator=g)
        self.offsets = torch.tensor(offsets, device="cuda")
        self.ids = torch.full((self.tokens,), -9, dtype=torch.int64, device="cuda")
        self.accepted = torch.full((len(rows),), -9, dtype=torch.int64, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        if not chance:
            self.draft = None

    def run(self, stream=None):
        sampling.Verifier(len(self.rows), self.tokens, self.vocab).verify(
            self.offsets, self.target, self.drafts, self.draft, self.accept, self.draw, self.ids, self.accepted,
            self.status, stream)

    def check(self, least=0.5):
        torch.cuda.synchronize()
        assert int(self.status) == 0
        host = lambda t: None if t is None else t.double().cpu().numpy()
        target, draft = host(self.target), host(self.draft)
        drafts, accept, draw = self.drafts.cpu().numpy(), host(self.accept), host(self.draw)
        ids, accepted, first, sure = self.ids.cpu().numpy(), self.accepted.cpu().numpy(), 0, 0
        for b, n in enumerate(self.rows):
            rows = slice(first, first + n)
            first += n
            if n == 0:
                assert accepted[b] == 0
                continue
            want, stop, margin = verify(n, target[rows], None if draft is None else draft[rows], drafts[rows],
                                        accept[rows], draw[b])
            assert accepted[b] == stop, b
            got = ids[rows].tolist()
            assert got[:stop] == want[:stop] and got[stop + 1:] == want[stop + 1:], b
            if margin > 1e-6:
                sure += 1
                assert got[stop] == want[stop], b
        assert sure >= least * len(self.rows)
        assert (ids[first:] == -9).all()  # rows of no request


@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 1024, 4099, 32768, 50257])
@pytest.mark.parametrize("rows", [[5], [1, 5, 3, 0, 2, 9, 1], [4] * 80], ids=["one", "ragged", "many"])
@pytest.mark.parametrize("chance", [True, False])
def test_verify_vs_float64(lib, cuda, rows, vocab, chance):
    for agree, filtered in ((0.3, False), (2.0, True)):
        d = Drafts(rows, vocab, seed=vocab, agree=agree, filtered=filtered, chance=chance)
        d.run()
        d.check()


def test_verify_large_vocabulary_and_many_drafts(lib, cuda):
    for rows, vocab in (([3, 2], 1 << 22), ([700, 1, 600], 515)):
        d = Drafts(rows, vocab, agree=0.02)
        d.run()
        # (a border every 2^-22 of the mass at the largest vocabulary)
        d.check(least=0.0 if vocab > 100000 else 0.5)


def test_verify_strides_and_alignment(lib, cuda):
    """Rows inside larger tensors at any alignment give the same tokens, and ids may be
    drafts."""
    d = Drafts([5, 2, 4], 5001, seed=4)
    d.run()
    d.check()
    ids, accepted = d.ids.clone(), d.accepted.clone()
    for off in (0, 1, 2, 3):
        wide = [torch.full((d.tokens, 5010 + off), math.nan, device="cuda") for _ in range(2)]
        for w, p in zip(wide, (d.target, d.draft)):
            w[:, off:off + 5001] = p
        e = Drafts([5, 2, 4], 5001, seed=4)
        e.target, e.draft = (w[:, off:off + 5001] for w in wide)
        if off == 1:
            e.ids = e.drafts
            kept = e.drafts[11:].clone()
        e.run()
        torch.cuda.synchronize()
        assert torch.equal(e.ids[:11], ids[:11]) and torch.equal(e.accepted, accepted)
        if off == 1:
            assert torch.equal(e.ids[11:], kept)


def test_verify_ends_of_the_ranges(lib, cuda):
    """Uniform numbers at and outside their ends, proposals outside the vocabulary, rows
    without mass, probabilities that are none."""
    nan, inf = math.nan, math.inf
    p = torch.tensor([[0.0, 0.5, 0.25, 0.25], [0.25, 0.25, 0.5, 0.0]], device="cuda")
    q = torch.tensor([[0.5, 0.25, 0.25, 0.0], [1.0, 0.0, 0.0, 0.0]], device="cuda")

    def one(x, u, w, target=p, draft=q):
        d = Drafts([2], 4, spare=0)
        d.target, d.draft = target.contiguous(), draft
        d.drafts = torch.tensor([x, 77], device="cuda")
        d.accept, d.draw = torch.tensor([u, nan], device="cuda"), torch.tensor([w], device="cuda")
        d.run()
        torch.cuda.synchronize()
        return d.ids.tolist() + d.accepted.tolist()

    assert one(1, 0.0, 0.0) == [1, 0, 1] and one(1, 0.999, 0.999) == [1, 2, 1]
    # a token of probability 0 is never accepted; max(p - q, 0) = [0, .25, 0, .25]
    assert one(0, 0.0, 0.0) == [1, -1, 0] and one(0, 0.0, 0.499) == [1, -1, 0]
    assert one(0, 0.0, 0.5) == [3, -1, 0] and one(0, 0.0, 0.999) == [3, -1, 0]
    for w in (1.0, 5.0, inf):
        assert one(0, 0.5, w) == [3, -1, 0]
    for w in (-1.0, nan):
        assert one(0, 0.5, w) == [1, -1, 0]
    assert one(1, nan, 0.0) == [1, -1, 0]  # a NaN accepts nothing
    # no proposal: from p itself
    for x in (-1, 4, 1 << 40, -(1 << 63)):
        assert one(x, 0.0, 0.0) == [1, -1, 0] and one(x, 0.0, 0.6) == [2, -1, 0]
    # made without chance: q is 1 at the proposal
    assert one(1, 0.499, 0.0, draft=None) == [1, 0, 1] and one(1, 0.5, 0.0, draft=None) == [2, -1, 0]
    # p <= q everywhere: from p; without mass: -1
    same = p.clone()
    assert one(0, 0.5, 0.6, draft=torch.maximum(p, q)) == [2, -1, 0]
    assert one(1, 1.0, 0.6, draft=same) == [2, -1, 0]
    assert one(1, 0.5, 0.5, target=torch.zeros(2, 4, device="cuda")) == [-1, -1, 0]
    # NaN and negative ones are 0, those above 1 are 1
    odd = torch.tensor([[nan, 7.0, -1.0, 0.5], [-inf, nan, inf, 0.0]], device="cuda")
    assert one(1, 0.999, 0.0, target=odd) == [1, 2, 1]
    assert one(0, 0.0, 0.0, target=odd) == [1, -1, 0] and one(0, 0.0, 0.999, target=odd) == [3, -1, 0]


def test_verify_bad_offsets(lib, cuda):
    d = Drafts([3, 2, 4], 200)
    d.offsets[1], d.offsets[3] = 9, 1 << 50  # falls after it, leaves the tensors
    d.run()
    torch.cuda.synchronize()
    assert int(d.status) == paged.BAD_OFFSET
    assert (d.accepted >= 0).all()


def test_verify_gives_the_targets_distribution(lib, cuda):
    """The first token that comes out is distributed as the target, whatever the draft: 4
    standard deviations over 200,000 requests with evenly spread numbers of their own."""
    n, vocab = 200000, 6
    g = torch.Generator(device="cuda").manual_seed(8)
    p = torch.tensor([0.3, 0.05, 0.15, 0.0, 0.4, 0.1], device="cuda")
    for q in (torch.tensor([0.1, 0.3, 0.15, 0.05, 0.1, 0.3], device="cuda"), p.clone()):
        d = Drafts([2] * n, vocab, spare=0)
        d.target = p.expand(2 * n, vocab).contiguous()
        d.draft = q.expand(2 * n, vocab).contiguous()
        d.drafts = torch.multinomial(q, 2 * n, replacement=True, generator=g)
        d.run()
        torch.cuda.synchronize()
        share = torch.bincount(d.ids[0::2], minlength=vocab).double() / n
        room = 4 * (p.double() * (1 - p.double()) / n).sqrt()
        assert ((share - p.double()).abs() <= room + 1e-12).all(), share


def test_verify_and_distributions_in_graphs_and_streams(lib, cuda):
    x = logits_of(9, 6000, BF16, 2)
    sampler, f = sampling.Sampler(9, 6000), filters(9, temperature=0.7, top_k=50)
    probs = torch.zeros(9, 6000, device="cuda")
    d = Drafts([5, 4], 6000, spare=0)
    v = sampling.Verifier(2, 9, 6000)
    side = torch.cuda.Stream()

    def both():
        sampler.probabilities(x, probs, **f)
        v.verify(d.offsets, probs, d.drafts, d.draft, d.accept, d.draw, d.ids, d.accepted, d.status)

    both()
    torch.cuda.synchronize()
    want = [t.clone() for t in (probs, d.ids, d.accepted)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        both()
    for t in (probs, d.ids, d.accepted):
        t.fill_(0)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((probs, d.ids, d.accepted), want))
    kept = x.clone()
    x.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):  # behind what the current stream holds
        torch.cuda._sleep(20_000_000)
        x.copy_(kept)
        both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((probs, d.ids, d.accepted), want))


def test_python_refusals(lib, cuda):
    s = sampling.Sampler(2, 10)
    x, p = torch.zeros(2, 10, device="cuda"), torch.zeros(2, 10, device="cuda")
    for args in ((x[:1], p), (x.double(), p), (x, p.half()), (x, p[:1]), (x, p.cpu()), (x, p.t().contiguous().t())):
        with pytest.raises(ValueError):
            s.probabilities(*args)
    with pytest.raises(ValueError):
        s.probabilities(x, p, top_p=torch.zeros(3, device="cuda"))
    d = Drafts([2, 1], 10, spare=0)
    good = [d.offsets, d.target, d.drafts, d.draft, d.accept, d.draw, d.ids, d.accepted]
    v = sampling.Verifier(2, 3, 10)
    for i in range(len(good)):
        for bad in (good[i].cpu(), good[i][:1], good[i].half()):
            with pytest.raises(ValueError):
                v.verify(*good[:i], bad, *good[i + 1:])
    with pytest.raises(ValueError):
        v.verify(*good, status=torch.zeros(2, dtype=torch.int32, device="cuda"))


# ---- together ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16])
def test_speculative_loop(lib, cuda, dtype):
    """Prompts, then steps of drafted tokens: append to the 8-bit cache, attend, project,
    distributions, verify, lengths from the accepted numbers, all on the device; the steps
    from a captured graph.  Every step's logits against float64 over the tokens that stood."""
    torch.manual_seed(5)
    vocab, heads, q_heads, dim, page, drafted = 300, 2, 4, 64, 16, 3
    prompts, steps = [37, 1, 64], 4
    n = drafted + 1
    emb = torch.randn(vocab, q_heads + 2 * heads, dim, device="cuda")
    head = torch.randn(q_heads * dim, vocab, device="cuda") * 0.2
    most = max(prompts) + steps * n + 1
    columns = -(-most // page)
    shape = (3 * columns, heads, page)
    pools = torch.zeros(2, *shape, dim, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(2, *shape, device="cuda")
    cache = paged.PagedCache8(pools[0], pools[1], scales[0], scales[1], dtype)
    table = torch.randperm(3 * columns, device="cuda").reshape(3, columns).int()
    rope = tuple(t.cuda() for t in rope_tables(most, dim))
    attend = paged.PagedAttention(cache, q_heads)
    first, sampler = sampling.Sampler(3, vocab), sampling.Sampler(3 * n, vocab)
    verifier = sampling.Verifier(3, 3 * n, vocab)
    text = [torch.randint(vocab, (m,), device="cuda") for m in prompts]
    lengths = torch.tensor(prompts, device="cuda")
    top_k = torch.full((3 * n,), 40, device="cuda")

    def pass_of(batch, flat):
        x = emb[flat].to(dtype)
        cache.append(batch, x[:, q_heads:q_heads + heads], x[:, q_heads + heads:], rope)
        o = torch.empty(flat.shape[0], q_heads, dim, dtype=dtype, device="cuda")
        attend.forward(batch, x[:, :q_heads], o, rope)
        return torch.matmul(o.flatten(1).float(), head)

    offsets = torch.tensor([0] + list(np.cumsum(prompts)), device="cuda")
    logits = pass_of(paged.PagedBatch(offsets, lengths, table, sum(prompts), 64), torch.cat(text))
    ids = torch.empty(3, dtype=torch.int64, device="cuda")
    first.sample(logits[offsets[1:] - 1].contiguous(), torch.rand(3, device="cuda"), ids, top_k=top_k[:3])
    text = [torch.cat([t, ids[b:b + 1]]) for b, t in enumerate(text)]

    rows = torch.arange(0, 3 * n + 1, n, device="cuda")
    batch = paged.PagedBatch(rows, lengths, table, 3 * n, n)
    flat = torch.empty(3 * n, dtype=torch.int64, device="cuda")
    drafts, draft = torch.empty_like(flat), torch.empty(3 * n, vocab, device="cuda")
    accept, uniform = torch.empty(3 * n, device="cuda"), torch.empty(3, device="cuda")
    seen, probs = torch.empty(3 * n, vocab, device="cuda"), torch.empty(3 * n, vocab, device="cuda")
    out, accepted = torch.empty_like(flat), torch.empty(3, dtype=torch.int64, device="cuda")

    def step():
        lengths.add_(n)  # the last token and the drafts behind it
        seen.copy_(pass_of(batch, flat))
        sampler.probabilities(seen, probs, top_k=top_k)
        verifier.verify(rows, probs, drafts, draft, accept, uniform, out, accepted)
        lengths.add_(accepted - drafted)  # what was not accepted is written over later

    side, graph, total = torch.cuda.Stream(), None, 0
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.matmul(torch.zeros(3 * n, q_heads * dim, device="cuda"), head)  # library set-up
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for t in range(steps):
        last = torch.stack([x[-1] for x in text])
        # a draft that often agrees: the last pass's logits with noise, or anything at first
        draft.copy_(torch.softmax(torch.randn(3 * n, vocab, device="cuda") * 2 + (seen if t else 0.0), 1))
        drafts.copy_(torch.multinomial(draft, 1)[:, 0])
        if t == 1:  # what the target itself finds likely is accepted
            drafts.view(3, n)[:, 0] = torch.stack([x[-1] for x in text])
        flat.copy_(torch.cat([last[:, None], drafts.view(3, n)[:, :drafted]], 1).flatten())
        accept.uniform_()
        uniform.uniform_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        host = [x.double().cpu().numpy() for x in (probs, draft, accept, uniform)]
        for b in range(3):
            own = slice(b * n, (b + 1) * n)
            want, stop, margin = verify(n, host[0][own], host[1][own], drafts[own].cpu().numpy(), host[2][own],
                                        host[3][b])
            assert int(accepted[b]) == stop
            assert margin <= 1e-6 or out[own].tolist() == want
            # the pass in float64 over the tokens that stood and this step's
            whole = torch.cat([text[b], drafts[own][:drafted]])
            m = whole.shape[0]
            x = emb[whole].to(dtype)
            k = rows_of(*quantise(turn_f32(x[:, q_heads:q_heads + heads], rope[0][:m], rope[1][:m])))
            v = rows_of(*quantise(x[:, q_heads + heads:].float()))
            q = turn(x[m - n:, :q_heads], rope[0][m - n:m], rope[1][m - n:m])
            o, _, weighted, spread = attention(q, k, v, m - n)
            u = 2.0 ** -11 if dtype == BF16 else 2.0 ** -20
            unit = 2.0 ** -8 if dtype == BF16 else 2.0 ** -24
            bound = ((2 * (u + 2.0 ** -16) * spread).expm1() + u + 2e-5)[..., None] * weighted + unit * o.abs()
            want = o.flatten(1) @ head.double()
            room = bound.flatten(1) @ head.double().abs() + 1e-4
            assert ((seen[own].double() - want).abs() <= room).all()
            total += stop
            text[b] = torch.cat([text[b], out[own][:stop + 1]])
            assert int(lengths[b]) == text[b].shape[0] - 1
