"""The serving operators at the ends of their ranges: magnitudes of scores and
values, masses far apart, infinite logits, metadata that leads outside, streams.

Tolerances.  An operand is off by p of its value: u = eps / 2 at f16 and bf16,
2^-22 at f32 (pairs of 22 bits), so a score by at most delta = (2 p + DIM 2^-23 +
2^-22) S, S = scale sum |q'||k| (both operands; the tensor pipe's accumulation;
the roundings of the score in f32 and of the base-2 exponential).  A weight is
then off by expm1(2 delta) relative, and o by that, its own and v's rounding (2 p)
and the sums' ((KEYS + 16) 2^-23; 2^-17 for exponentials by polynomial), all of
sum p|v|, plus its last rounding u |o|.
"""
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from eshkol_transformer_b200 import build, paged, sampling
from serving_f64 import attention, sample, turn
from test_gpu_serving import BF16, F16, F32, U, Step, draw

pytestmark = pytest.mark.gpu


def run(s, hint, rope=True):
    """s.o, s.lse by the kernel of few (hint 1) or many (100) rows."""
    b = paged.PagedBatch(s.offsets, s.lengths, s.table, s.tokens, hint, None, s.status)
    s.o.fill_(7.0)
    s.lse.fill_(7.0)
    paged.PagedAttention(s.cache, s.q_heads).forward(b, s.q, s.o, (s.cos, s.sin) if rope else None,
                                                     s.lse)
    torch.cuda.synchronize()
    assert int(s.status) == 0


def expected(s, rope=True):
    """(rows, keys, o, lse, weighted |v|, largest S) of each request, in float64."""
    first = 0
    for b, (n, m) in enumerate(s.requests):
        rows = slice(first, first + n)
        first += n
        q = s.q[rows].double()
        if rope:
            q = turn(q, s.cos[m - n:m], s.sin[m - n:m])
        yield (rows, m, *attention(q, s.k[b].double(), s.v[b].double(), m - n))


def check(s, rope=True):
    p = {F32: 2.0 ** -22}.get(s.dtype, U[s.dtype])
    for rows, m, o, lse, weighted, spread in expected(s, rope):
        delta = (2 * p + s.q.shape[-1] * 2.0 ** -23 + 2.0 ** -22) * spread
        wide = (2 * delta).expm1() + 2 * p + (m + 16) * 2.0 ** -23 + 2.0 ** -17
        bound = wide[..., None] * weighted + U[s.dtype] * o.abs() + 1e-30
        over = (s.o[rows].double() - o).abs() - bound
        assert (over <= 0).all(), float(over.max())
        assert ((s.lse[rows].double() - lse).abs() <= delta + 2e-5 * (1 + lse.abs())).all()


@pytest.mark.parametrize("scale", [30.0, 1000.0, 4000.0])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hint", [1, 100])
def test_f32_scores_in_the_thousands(lib, cuda, hint, dim, scale):
    """Scores of +-3 to +-12,000, where neighbouring bfloat16 numbers lie up to 64
    apart: the probabilities stand on the row's maximum itself."""
    s = Step([(40, 300), (1, 500), (130, 700)], 2, 1, dim, 16, F32, seed=dim)
    s.q *= scale
    run(s, hint)
    check(s)


ZERO, HUGE = -1000, 47


def value_rows(pattern, m, g):
    """Exponents of the m rows of values."""
    at = torch.arange(m, device="cuda")
    some = torch.randint(0, 3, (m,), device="cuda", generator=g) == 0
    if pattern == "one huge":
        return torch.where(at == 3, HUGE, ZERO)
    if pattern == "half huge":
        return torch.where(some, HUGE, ZERO)
    if pattern == "late huge":
        return torch.where((at > m // 2) & some, HUGE, ZERO)
    if pattern == "early huge":
        return torch.where((at < m // 4) & some, HUGE, ZERO)
    if pattern == "largest and ones":
        return torch.where(some, 110, torch.where(at % 5 == 0, ZERO, 0))
    if pattern == "any":
        return torch.randint(-100, 101, (m,), device="cuda", generator=g)
    if pattern == "small":
        return torch.where(some, -70, ZERO)
    return torch.full((m,), ZERO, device="cuda")  # "zeros"


@pytest.mark.parametrize("requests", [[(40, 700), (150, 150)], [(20, 9001)]], ids=["blocks", "joined"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("scores", ["equal", "normal"])
@pytest.mark.parametrize("pattern", ["one huge", "half huge", "late huge", "early huge",
                                     "largest and ones", "any", "small", "zeros"])
def test_f32_value_rows_of_any_magnitude(lib, cuda, pattern, scores, dim, requests):
    """Rows of zeros and rows up to 2^110 next to one another: each keeps its share
    of the denominator.  (With rows of 0 and 2^47 at equal scores the output is their
    mean.)"""
    s = Step(requests, 2, 1, dim, 16, F32, seed=dim)
    g = torch.Generator(device="cuda").manual_seed(dim)
    if scores == "equal":
        s.q.zero_()
    for b, (_, m) in enumerate(requests):
        e = value_rows(pattern, m, g)
        s.v[b] *= torch.where(e == ZERO, 0.0, torch.exp2(e.float()))[:, None, None]
        s.store(b, s.k[b], s.v[b])
    for hint in (1, 100):
        run(s, hint)
        for rows, m, o, lse, weighted, _ in expected(s):
            room = 2e-5 * weighted.amax(-1, keepdim=True)
            assert ((s.o[rows].double() - o).abs() <= room).all(), hint
            assert ((s.lse[rows].double() - lse).abs() <= 2e-5 * (1 + lse.abs())).all(), hint


@pytest.mark.parametrize("dim", [64, 128])
def test_f32_far_value_behind_a_low_score(lib, cuda, dim):
    """A key whose value is 2^100 and whose weight is below 2^-400 changes nothing."""
    s = Step([(40, 700)], 2, 1, dim, 16, F32, seed=dim)
    s.q.copy_(s.q[:1, :1].expand_as(s.q).clone())
    s.k[0][5] = -40.0 * s.q[0, :1]
    s.v[0][5] *= 2.0 ** 100
    s.store(0, s.k[0], s.v[0])
    for hint in (1, 100):
        run(s, hint, rope=False)
        for rows, m, o, lse, _, _ in expected(s, rope=False):
            assert ((s.o[rows].double() - o).abs() <= 2e-5 * (1 + o.abs())).all(), hint
            assert ((s.lse[rows].double() - lse).abs() <= 2e-5 * (1 + lse.abs())).all(), hint


@pytest.mark.parametrize("dim", [64, 128])
def test_f32_many_zero_values(lib, cuda, dim):
    """20,000 keys with values of zero, the first ones a little less likely: the sum
    of weights stays inside f32.  150 requests share the pages, so that a thread
    block has all keys of one."""
    new, length, page, batch = 20, 20000, 16, 150
    keys = torch.zeros(length // page, 1, page, dim, device="cuda")
    keys[:4] = -5.4 / math.sqrt(dim)  # e^-5.4 of the others' weight
    cache = paged.PagedCache(keys, torch.zeros_like(keys))
    table = torch.arange(length // page, device="cuda").int().expand(batch, -1).contiguous()
    offsets = torch.arange(batch + 1, device="cuda") * new
    q = torch.ones(batch * new, 1, dim, device="cuda")
    seen = length - new + 1 + torch.arange(new, device="cuda").double()
    want = torch.log((seen - 64) + 64 * math.exp(-5.4)).repeat(batch)
    for hint in (1, new):
        o, lse = torch.full_like(q, 7.0), torch.full((batch * new, 1), 7.0, device="cuda")
        b = paged.PagedBatch(offsets, torch.full((batch,), length, device="cuda"), table, batch * new, hint)
        paged.PagedAttention(cache, 1).forward(b, q, o, None, lse)
        torch.cuda.synchronize()
        assert (o == 0).all() and ((lse[:, 0].double() - want).abs() <= 2e-4).all(), hint


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("hint", [1, 100])
@pytest.mark.parametrize("gap", [12.0, 16.5])
def test_many_unlikely_keys_behind_a_likely_one(lib, cuda, gap, hint, dim, dtype):
    """One key without a value takes nearly all weight (an attention sink), 4,000
    others, e^-gap each, carry the output: their weights keep their bits.  (32 heads, so
    that a thread block walks many keys behind the likely one.)  The scores' products
    are exact: what is left are the weights' rounding u, the exponentials' 2^-18 (by
    polynomial; 2^-20 of f32 scores of 24) and sums' (KEYS + 16) 2^-23, and the
    output's rounding, absolute below the normal range."""
    s = Step([(20, 4001)], 32, 32, dim, 16, dtype, seed=dim)
    s.q.fill_(1.0)
    s.k[0].zero_()
    s.k[0][7] = gap / math.sqrt(dim)
    s.v[0] += 1.0
    s.v[0][7] = 0.0
    s.store(0, s.k[0], s.v[0])
    run(s, hint, rope=False)
    u = U[dtype]
    for rows, m, o, lse, weighted, _ in expected(s, rope=False):
        bound = (u + 2.0 ** -17 + (m + 16) * 2.0 ** -23) * weighted + u * o.abs()
        bound += torch.finfo(dtype).smallest_normal * u
        assert ((s.o[rows].double() - o).abs() <= 1.01 * bound).all()
        assert ((s.lse[rows].double() - lse).abs() <= 2e-5 * (1 + lse.abs())).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("hint", [1, 100])
def test_f16_queries_near_the_largest(lib, cuda, hint, dim):
    """Queries of up to 65,000 whose rotation passes 65,504, the largest f16."""
    s = Step([(30, 200), (1, 77)], 2, 1, dim, 16, F16, seed=dim)
    s.q.copy_(65000.0 * (1.0 - 0.2 * s.q.float().abs().clamp(max=4.0)))
    assert float(turn(s.q[29:30].double(), s.cos[[199]], s.sin[[199]]).abs().max()) > 70000.0
    for b in range(2):
        s.k[b] *= 2.0 ** -13
        s.store(b, s.k[b], s.v[b])
    run(s, hint)
    check(s)


@pytest.mark.parametrize("vocab", [7, 900, 4099, 30011])
def test_sampling_infinite_temperature(lib, cuda, vocab):
    """Every logit above -inf weighs the same, and every row gets an answer."""
    x = torch.randn(16, vocab, device="cuda")
    x[:, 1::3] = -math.inf
    some = np.nonzero((x[0] > -math.inf).cpu().numpy())[0]
    u = ((np.arange(16) + 0.5) / 16).astype(np.float32)
    for kw in (dict(), dict(min_p=1.0), dict(min_p=0.3), dict(min_p=5.0), dict(top_p=1.0, min_p=1.0)):
        ids, lp = draw(x, u, math.inf, **kw)
        assert np.array_equal(ids, some[np.floor(u.astype(np.float64) * some.size).astype(int)]), kw
        assert np.allclose(lp, -math.log(some.size), atol=2e-6), kw
    for kw, left in ((dict(top_k=4), 4), (dict(top_k=4, min_p=1.0), 4),
                     (dict(top_k=4, top_p=0.75, min_p=0.5), 3)):
        ids, lp = draw(x, u, math.inf, **kw)
        for r in range(16):
            kept = np.sort(np.argsort(-x[r].double().cpu().numpy(), kind="stable")[:left])
            assert ids[r] == kept[int(u[r] * left)] and abs(lp[r] + math.log(left)) <= 2e-6, kw


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [5, 2000])
def test_sampling_logits_further_apart_than_the_largest_f32(lib, cuda, vocab, dtype):
    """max x - x overflows f32, the weight exp((x - max x) / temperature) does not."""
    x = torch.full((3, vocab), -3.3e38, device="cuda")
    x[:, 1], x[:, 3] = 3.3e38, 0.0
    x = x.to(dtype)
    host = x[0].double().cpu().numpy()
    for t in (math.inf, 3e38, 1e37, 1.0):
        for kw in (dict(), dict(top_p=0.9), dict(min_p=0.3), dict(top_k=3)):
            u = np.array([0.0, 0.37, 0.93], np.float32)
            ids, lp = draw(x, u, t, **kw)
            for r in range(3):
                i, want, room = sample(host, float(u[r]), float(np.float32(t)), kw.get("top_k", 0),
                                       float(np.float32(kw.get("top_p", 1.0))),
                                       float(np.float32(kw.get("min_p", 0.0))))
                assert room <= 2.5e-7 or (ids[r] == i and abs(lp[r] - want) <= 2e-6), (t, kw, r)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [900, 5000, 30011, 300001])
def test_sampling_infinite_logits_among_many(lib, cuda, vocab, dtype):
    """+inf logits share all weight whatever the filters, also where cuts come from
    histograms over the logits."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(4, vocab, device="cuda", generator=g).to(dtype)
    x[:, 5:9] = math.nan
    x[:, 20:40] = -math.inf
    where = [3, 17, vocab // 2, vocab - 2, vocab - 1]
    for r in range(4):
        x[r, where[:r + 1]] = math.inf
    u = np.array([0.7, 0.45, 0.6, 0.95], np.float32)
    for kw in (dict(), dict(top_p=0.9), dict(top_p=0.5), dict(min_p=0.2), dict(top_k=2),
               dict(top_k=600), dict(top_k=600, top_p=0.8, min_p=0.1)):
        ids, lp = draw(x, u, 0.7, **kw)
        for r in range(4):
            i, want, _ = sample(x[r].double().cpu().numpy(), float(u[r]), 0.7, kw.get("top_k", 0),
                                kw.get("top_p", 1.0), kw.get("min_p", 0.0))
            assert ids[r] == i and abs(lp[r] - want) <= 2e-6, (r, kw)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("vocab", [200001, 300001, 425968, 450001])
def test_sampling_draws_inside_a_likely_token(lib, cuda, vocab, dtype):
    """Slices that fill a cluster's shared memory and vocabularies beyond them, each
    draw in the middle of a likely token's share."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(6, vocab, device="cuda", generator=g)
    likely = torch.randint(vocab, (6, 8), device="cuda", generator=g)
    x.scatter_(1, likely, 15.0 + 0.25 * torch.arange(8, device="cuda").expand(6, 8))
    x = x.to(dtype)
    host = x.double().cpu().numpy()
    for kw in (dict(), dict(top_k=64), dict(top_p=0.5), dict(min_p=0.3), dict(top_k=1000, top_p=0.9),
               dict(top_p=0.97)):
        u, want = np.zeros(6, np.float32), []
        for r in range(6):
            args = kw.get("top_k", 0), kw.get("top_p", 1.0), kw.get("min_p", 0.0)
            # the middle of the likeliest token's share of what the filters keep
            best = int(host[r].argmax())
            order = np.lexsort((np.arange(vocab), -host[r]))
            w = np.exp(host[r][order] - host[r].max())
            if args[0]:
                w[args[0]:] = 0.0
            before = np.cumsum(w) - w
            w[(before >= args[1] * w.sum()) & (args[1] < 1.0)] = 0.0
            w[w < args[2]] = 0.0
            run_sum = np.zeros(vocab)
            run_sum[order] = w
            run_sum = np.cumsum(run_sum)
            u[r] = (run_sum[best] - 0.5) / run_sum[-1]  # its weight is 1
            i, lp, _ = sample(host[r], float(u[r]), 1.0, *args)
            assert i == best
            want.append(lp)
        ids, lp = draw(x, u, 1.0, **kw)
        assert np.array_equal(ids, host.argmax(1)), kw
        assert np.allclose(lp, want, atol=2e-6), kw


def test_waits_that_run_out_are_reported(cuda, tmp_path):
    """From any warp, with and without a status word (see paged_wait.cu)."""
    root, out = Path(__file__).resolve().parents[1], tmp_path / "paged_wait"
    subprocess.run([build.nvcc(), *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr",
                    f"-I{build.INCLUDE}", f"-I{build.CSRC}", str(root / "tests" / "paged_wait.cu"),
                    "-o", str(out)], check=True)
    done = subprocess.run([str(out)], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and done.stdout.strip() == "ok", done.stdout


def test_append_records_every_request(lib, cuda):
    """What is wrong with a request is recorded whether or not a token of it is
    stored, as the attention does."""
    for change, bit in (((("offsets", 2, 99),), paged.BAD_OFFSET), ((("offsets", 0, -3),), paged.BAD_OFFSET),
                        ((("lengths", 1, 1 << 40),), paged.BAD_LENGTH),
                        ((("lengths", 1, -1),), paged.BAD_LENGTH), ((), 0)):
        for many in (0, 3000):  # requests behind the two, without tokens
            s = Step([(2, 20), (0, 9)] + [(0, 0)] * many, 2, 1, 64, 16, F16, spare=0)
            for name, i, x in change:
                getattr(s, name)[i if i < 2 else -1] = x
            k = torch.zeros(2, 1, 64, dtype=F16, device="cuda")
            s.cache.append(s.batch(), k, k)
            torch.cuda.synchronize()
            assert int(s.status) == bit, (change, many)
            s.status.zero_()
            s.attend()
            torch.cuda.synchronize()
            assert int(s.status) == bit, (change, many)


def test_calls_follow_the_current_stream(lib, cuda):
    """Without `stream` a call takes torch's current one: it comes after what was
    enqueued there, and into a capture."""
    s = Step([(1, 40), (3, 30)], 2, 1, 64, 16, F16, spare=0)
    a = paged.PagedAttention(s.cache, 2)
    sampler = sampling.Sampler(4, 5000)
    logits, ids = torch.zeros(4, 5000, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    u = torch.zeros(4, device="cuda")
    k, v = torch.randn(2, s.tokens, 1, 64, device="cuda").half()
    q, batch = torch.zeros_like(s.q), s.batch()
    keys, values = s.keys.clone().nan_to_num(), s.values.clone().nan_to_num()
    s.keys.nan_to_num_()
    s.values.nan_to_num_()

    def step():
        s.cache.append(batch, k, v, rope=(s.cos, s.sin))
        a.forward(batch, q, s.o, (s.cos, s.sin), s.lse)
        sampler.sample(logits, u, ids)

    q.copy_(s.q)
    logits[:, 77] = 100.0
    step()
    torch.cuda.synchronize()
    want = [t.clone() for t in (s.o, s.keys, ids)]
    for t in (q, s.o, s.lse, logits, ids):
        t.zero_()
    s.keys.copy_(keys)
    s.values.copy_(values)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # what follows has to wait for this
        q.copy_(s.q)
        logits[:, 77] = 100.0
        step()
    side.synchronize()
    for now, then in zip((s.o, s.keys, ids), want):
        assert torch.equal(now, then)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    s.o.zero_()
    ids.zero_()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(s.o, want[0]) and torch.equal(ids, want[2])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (64, 24), (80, 7), (256, 8)])
@pytest.mark.parametrize("hint", [1, 100])
def test_bad_metadata_of_every_kernel(lib, cuda, hint, dim, page, dtype):
    """Pages outside the pool read as zeros; lengths, offsets and positions beyond
    the tables are clamped: in the kernels of few and of many rows, with pages
    copied by TMA and one by one."""
    s = Step([(1, 40), (20, 400), (1, 20)], 2, 1, dim, page, dtype)
    s.keys.nan_to_num_()
    s.values.nan_to_num_()
    for what, bit in (("page", paged.BAD_PAGE), ("length", paged.BAD_LENGTH),
                      ("offset", paged.BAD_OFFSET), ("rope", paged.BAD_ROPE)):
        keep = [t.clone() for t in (s.table, s.lengths, s.offsets)]
        rope = (s.cos, s.sin)
        if what == "page":
            s.table[0, 0], s.table[1, 1], s.table[2, 0] = -1, s.keys.shape[0], 2 ** 31 - 1
        elif what == "length":
            s.lengths[0], s.lengths[1] = -(2 ** 40), 2 ** 40
        elif what == "offset":
            s.offsets[1], s.offsets[3] = 2 ** 40, -9
        else:
            rope = (s.cos[:3].contiguous(), s.sin[:3].contiguous())
        s.status.zero_()
        s.o.fill_(7.0)
        b = paged.PagedBatch(s.offsets, s.lengths, s.table, s.tokens, hint, None, s.status)
        paged.PagedAttention(s.cache, 2).forward(b, s.q, s.o, rope, s.lse)
        torch.cuda.synchronize()
        assert int(s.status) & bit, what
        assert torch.isfinite(s.o.float()).all()
        if what == "page":  # as with pages of zeros in their place
            s.status.zero_()
            for r, c in ((0, 0), (1, 1), (2, 0)):
                s.table[r, c] = keep[0][r, c]
                for b_, t in ((r, s.k), (r, s.v)):
                    t[b_][c * page:(c + 1) * page] = 0.0
                s.store(r, s.k[r], s.v[r])
            got = s.o.clone()
            run(s, hint)
            assert torch.equal(s.o[:s.used], got[:s.used])
        for t, old in zip((s.table, s.lengths, s.offsets), keep):
            t.copy_(old)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("page", [16, 24])
def test_captured_chunks(lib, cuda, page, dtype):
    """Captured steps of many rows, two graphs with their own workspaces side by
    side: the same bits as the eager call, replay after replay."""
    steps = [Step([(70, 700), (1, 90), (33, 2000)], 4, 2, 64, page, dtype, seed=i) for i in range(2)]
    objects = [paged.PagedAttention(s.cache, 4) for s in steps]
    graphs, streams, batches = [], [torch.cuda.Stream() for _ in steps], [s.batch() for s in steps]
    for s, a, b, stream in zip(steps, objects, batches, streams):
        s.attend(attention_object=a)
        s.check()
        s.first = s.o.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            a.forward(b, s.q, s.o, (s.cos, s.sin), s.lse, stream=stream.cuda_stream)
        graphs.append(graph)
        s.o.fill_(7.0)
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for s in steps:
        assert torch.equal(s.o, s.first)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_more_requests_than_threads(lib, cuda, dtype):
    """700 requests, a few of them with many rows: the division takes several
    passes in the kernels of many rows too."""
    s = Step([(40 if b % 300 == 7 else b % 2, 1 + 7 * b % 130 + 40) for b in range(700)], 2, 1, 64, 16,
             dtype, seed=4)
    for hint in (1, 100):
        run(s, hint)
        s.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,page,dim", [(2, 16, 64), (1, 8, 128), (3, 1, 64), (1, 1, 32), (2, 24, 40)])
@pytest.mark.parametrize("hint", [1, 100])
def test_pools_inside_a_larger_tensor(lib, cuda, hint, heads, page, dim, dtype):
    """Keys and values of one layer of a [pages, layers, 2, ...] tensor, appended and
    attended in place; the other layers stay as they are."""
    s = Step([(1, 40), (20, 90), (3, 3)], 2 * heads, heads, dim, page, dtype)
    pages = s.keys.shape[0]
    for layout in ("heads", "slots"):
        shape = (heads, page, dim) if layout == "heads" else (page, heads, dim)
        whole = torch.full((pages, 3, 2, *shape), 5.0, dtype=dtype, device="cuda")
        s.keys, s.values = whole[:, 1, 0], whole[:, 1, 1]
        if layout == "slots":
            s.keys, s.values = s.keys.transpose(1, 2), s.values.transpose(1, 2)
        s.cache = paged.PagedCache(s.keys, s.values)
        new = [torch.cat([t[b][m - n:] for b, (n, m) in enumerate(s.requests)] + [t[0][:2]])
               for t in (s.k, s.v)]
        for b, (n, m) in enumerate(s.requests):  # what was cached before this step
            s.store(b, s.k[b][:m - n], s.v[b][:m - n])
        s.cache.append(s.batch(), *new)
        run(s, hint)
        check(s)
        assert (whole[:, 0] == 5.0).all() and (whole[:, 2] == 5.0).all()


def test_two_host_threads(lib, cuda):
    """Steps issued from two threads on streams of their own, each with its own
    objects, give the bits that they give alone."""
    import threading
    steps = [Step([(1, 900), (30, 300)], 4, 2, 64, 16, t, seed=i) for i, t in enumerate((F16, F32))]
    want, streams, errors = [], [torch.cuda.Stream() for _ in steps], []
    for s in steps:
        s.attend()
        s.check()
        want.append(s.o.clone())
        s.o.fill_(7.0)
    torch.cuda.synchronize()

    def work(s, stream, first):
        try:
            a = paged.PagedAttention(s.cache, s.q_heads)
            x = torch.zeros(2, 5000, device="cuda")
            ids = torch.full((2,), -7, dtype=torch.int64, device="cuda")
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                for _ in range(50):
                    s.attend(attention_object=a, stream=None)
                    sampling.Sampler(2, 5000).sample(x, x[:, 0].contiguous(), ids)
            stream.synchronize()
            assert torch.equal(s.o, first) and (ids == 0).all()
        except BaseException as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(steps, streams, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
