"""The 8-bit paged cache (quantising append, attention over it) against the definition in
float64.

Tolerances.  Append: the elements and scales are those of the rotated row in f32, whose
four operations round one by one, so bytes and scales are equal.  Attention: an element and
its scale are exact, and q' and the weights are binary16 (u = 2^-11): a score is off by at
most delta = (u + DIM 2^-23) scale sum |q'||k| + 2^-22 |score| (f32 accumulation, the
base-2 exponential), a weight by exp(2 delta) - 1 relative and by u for its own rounding;
exponentials by polynomial are off by 2.7e-6, in numerator and denominator (2^-17
together); weights are multiples of 2^-38 of the row's largest weight times value scale,
which 2^-17 covers too; then u of the output's type (f16 below 2^-14 is spaced 2^-24: off by
up to 2^-25 whatever the value).  At f32 the bar of the framework's
other f32-grade attention tests: 2e-5 absolute plus relative.
"""
import math
import threading

import pytest
import torch

from cache8_f64 import quantise, rows_of, turn_f32
from eshkol_transformer_b200 import paged
from serving_f64 import attention, ragged, rope_tables, turn

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


class Step8:
    """An 8-bit cache and one step's tensors.  Bytes and scales are NaN wherever no
    request keeps a key; `spare` rows follow the last request's."""

    def __init__(self, requests, q_heads, heads, dim, page, dtype, seed=1, layout="heads", spare=2,
                 strided=False, loose_scales=False, sizes=None, scale_factor=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
        self.requests, self.dtype, self.page, self.heads, self.dim = requests, dtype, page, heads, dim
        offsets, lengths = ragged(requests)
        self.offsets = torch.tensor(offsets, device="cuda")
        self.lengths = torch.tensor(lengths, device="cuda")
        self.used, self.tokens = offsets[-1], offsets[-1] + spare
        longest = max(lengths + [1])
        columns, batch = -(-longest // page), len(requests)
        pages = batch * columns + 2
        self.table = torch.randperm(pages, device="cuda", generator=g)[:batch * columns]
        self.table = self.table.reshape(batch, columns).int()
        first = layout == "heads"
        shape = (pages, heads, page) if first else (pages, page, heads)
        pools = [torch.full(shape + (dim,), 0x7f, device="cuda", dtype=torch.uint8) for _ in range(2)]
        every = 3 if loose_scales else 1
        scales = [torch.full(shape + (every,), math.nan, device="cuda")[..., 0] for _ in range(2)]
        turned = lambda t: t if first else t.transpose(1, 2)
        self.keys, self.values = [turned(p) for p in pools]
        self.key_scales, self.value_scales = [turned(p) for p in scales]
        # every key and value of the requests, rows of differing sizes, as the cache has them
        self.k, self.v = [], []
        for b, (_, m) in enumerate(requests):
            for pool, scale, rows in ((self.keys, self.key_scales, self.k),
                                      (self.values, self.value_scales, self.v)):
                x = rand(m, heads, dim) * (0.5 * rand(m, heads, 1)).exp()
                if sizes is not None:
                    x = x * sizes(m, heads, g)
                bits, s = quantise(x.float())
                s = s * scale_factor
                where, slot = self.slots(b, 0, m)
                pool[where, :, slot] = bits
                scale[where, :, slot] = s
                rows.append(rows_of(bits, s))
        width = q_heads * dim + (3 if strided else 0)
        self.q = rand(self.tokens, width).to(dtype)[:, width - q_heads * dim:].unflatten(1, (q_heads, dim))
        self.o = torch.full((self.tokens, width), 7.0, device="cuda", dtype=dtype)
        self.o = self.o[:, width - q_heads * dim:].unflatten(1, (q_heads, dim))
        self.lse = torch.full((self.tokens, q_heads), 7.0, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.cos, self.sin = [t.cuda() for t in rope_tables(longest, dim)]
        self.cache = paged.PagedCache8(self.keys, self.values, self.key_scales, self.value_scales, dtype)
        self.q_heads = q_heads

    def slots(self, b, first, last):
        at = torch.arange(first, last, device="cuda")
        return self.table[b].long()[at // self.page], at % self.page

    def batch(self, max_new=None):
        most = max((n for n, _ in self.requests), default=0) if max_new is None else max_new
        return paged.PagedBatch(self.offsets, self.lengths, self.table, self.tokens, most, None, self.status)

    def attend(self, rope=True, stream=None, attention_object=None, max_new=None):
        a = attention_object or paged.PagedAttention(self.cache, self.q_heads)
        a.forward(self.batch(max_new), self.q, self.o, (self.cos, self.sin) if rope else None, self.lse, stream)

    def check(self, rope=True, f32_bar=2e-5, status=0):
        torch.cuda.synchronize()
        assert int(self.status) == status
        first = 0
        for b, (n, m) in enumerate(self.requests):
            rows = slice(first, first + n)
            first += n
            if n == 0:
                continue
            at = torch.arange(m - n, m, device="cuda").clamp_min(0)
            q = self.q[rows].double()
            if rope and m > 0:
                q = turn(q, self.cos[at], self.sin[at])
            o, lse, weighted, spread = attention(q, self.k[b], self.v[b], m - n)
            got, dim = self.o[rows].double(), q.shape[-1]
            if self.dtype == F32:
                bound = f32_bar * (1 + o.abs()) if f32_bar == 2e-5 else f32_bar * weighted.amax(-1, keepdim=True)
                lse_bound = 2e-5 + 2e-5 * lse.abs()
            else:
                u = 2.0 ** -11
                delta = (u + dim * 2.0 ** -23) * spread + 2.0 ** -22 * spread
                wide = (2 * delta).expm1() + u + (m + 16) * 2.0 ** -23 + 2.0 ** -17
                least = 2.0 ** -25 if self.dtype == F16 else 1e-30
                bound = wide[..., None] * weighted + U[self.dtype] * o.abs() + least
                lse_bound = delta + 2e-5 * (1 + lse.abs())
            empty = torch.isinf(lse)
            assert torch.equal(torch.isinf(self.lse[rows]), empty)
            assert (got[empty] == 0).all()
            assert ((got - o).abs() <= bound).all(), (b, float(((got - o).abs() - bound).max()))
            assert ((self.lse[rows].double() - lse).abs() <= lse_bound)[~empty].all()
        # rows of no request stay as they were
        assert (self.o[self.used:] == 7.0).all() and (self.lse[self.used:] == 7.0).all()


# ---- append ---------------------------------------------------------------------------------

def pools_of(s):
    return [s.keys, s.values, s.key_scales, s.value_scales]


def appended(s, k, v, rope=True):
    """The pools after the append of s's new tokens, by definition."""
    want = [p.clone() for p in pools_of(s)]
    first = 0
    for b, (n, m) in enumerate(s.requests):
        rows = slice(first, first + n)
        first += n
        skip = max(0, n - m)  # tokens at negative positions are not stored
        if n - skip <= 0:
            continue
        at = torch.arange(m - n + skip, m, device="cuda")
        kr, vr = k[rows][skip:], v[rows][skip:].float()
        kr = turn_f32(kr, s.cos[at], s.sin[at]) if rope else kr.float()
        where, slot = s.slots(b, m - n + skip, m)
        for i, x in enumerate((kr, vr)):
            want[i][where, :, slot], want[i + 2][where, :, slot] = quantise(x)
    return want


def same(a, b):
    """Equal, NaN where NaN."""
    if a.dtype == torch.uint8:
        return torch.equal(a, b)
    return torch.equal(torch.nan_to_num(a, nan=-1.0), torch.nan_to_num(b, nan=-1.0))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,dim,page,layout,strided", [
    (1, 16, 1, "heads", False), (4, 64, 16, "heads", False), (3, 80, 24, "slots", True),
    (8, 128, 16, "slots", False), (16, 128, 64, "heads", True), (5, 256, 8, "heads", False),
    (2, 48, 7, "heads", True), (40, 32, 16, "heads", False)])
def test_append(lib, cuda, heads, dim, page, layout, strided, dtype):
    s = Step8([(5, 40), (0, 3), (1, 1), (33, 33), (4, 2), (0, 0), (130, 700)], heads, heads, dim, page, dtype,
              seed=dim, layout=layout)
    width = heads * dim + (3 if strided else 0)
    k, v = (torch.randn(s.tokens, width, device="cuda").to(dtype)[:, width - heads * dim:].unflatten(1, (heads, dim))
            for _ in range(2))
    k[7], v[2] = 0.0, 0.0
    for rope in (True, False):
        want = appended(s, k, v, rope)
        s.cache.append(s.batch(), k, v, (s.cos, s.sin) if rope else None)
        torch.cuda.synchronize()
        assert int(s.status) == 0
        for got, w in zip(pools_of(s), want):
            assert same(got, w)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_of_extreme_rows(lib, cuda, dtype):
    """Rows at the ends of the type's range, at the borders of a scale, of zeros and with
    infinities and NaN."""
    s = Step8([(40, 40)], 2, 2, 64, 16, dtype, spare=0)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(40, 2, 64, device="cuda", generator=g)
    x = (x * torch.exp2(torch.arange(40, device="cuda").float() * 6 - 120)[:, None, None]).to(dtype)
    for i, top in enumerate((448.0, 449.0, 450.0, 447.0, 1.75, 1.7578125, 3.5, 2.0 ** -149, 2.0 ** -126, 3.38e38)):
        x[i] = x[i].float().clamp(-0.5, 0.5).to(dtype) * 0
        x[i, :, 3], x[i, :, 9] = top, -top / 3
    x[20, 0] = 0.0
    x[21, 1, 5], x[22, 0, 63], x[23, 0, 0] = math.inf, math.nan, -math.inf
    v = x.flip(0).contiguous()
    want = appended(s, x, v, False)
    s.cache.append(s.batch(), x, v)
    torch.cuda.synchronize()
    sound = ~torch.isnan(want[2])
    assert same(s.key_scales, want[2]) and same(s.value_scales, want[3])
    assert int(torch.isnan(s.key_scales[s.table[0].long()]).sum()) >= 3
    assert torch.equal(s.keys[sound], want[0][sound])
    ok = ~torch.isnan(want[3])
    assert torch.equal(s.values[ok], want[1][ok])
    # such a row makes NaN of what sees it
    s.attend(rope=False)
    torch.cuda.synchronize()
    assert torch.isnan(s.o[39].float()).any()


@pytest.mark.parametrize("dtype,n,m,q_heads,heads,dim,page", [
    (F32, 1, 300, 4, 2, 64, 16), (BF16, 1, 5000, 16, 2, 128, 64), (F16, 5, 700, 6, 2, 80, 24),
    (BF16, 12, 900, 4, 2, 256, 16), (F16, 40, 900, 6, 3, 256, 16), (F32, 60, 400, 4, 2, 128, 16),
    (BF16, 200, 1500, 4, 2, 128, 16), (F16, 300, 300, 8, 2, 64, 8), (F32, 150, 700, 4, 2, 64, 32),
    (BF16, 200, 500, 4, 2, 128, 24)])
@pytest.mark.parametrize("where", ["new", "old"])
def test_rows_that_are_not_finite_reach_the_queries_that_see_them_alone(lib, cuda, dtype, n, m, q_heads,
                                                                        heads, dim, page, where):
    """One row of keys, another of values, of head 0 that hold an infinity or a NaN: NaN for the
    queries of that head from the first of their positions on, nothing for all others."""
    s = Step8([(n, m)], q_heads, heads, dim, page, dtype, spare=0)
    s.attend()
    sound = s.o.clone().double()
    # positions 6 and 7 of eight, where exponentials may take another pipe
    first = m - 1 if where == "new" and n == 1 else m - n // 2 if where == "new" else (m - n) // 2 // 8 * 8 + 6
    if where == "old" and m == n:
        first = 6
    bad = Step8([(n, m)], q_heads, heads, dim, page, dtype, spare=0)
    # a step that stores non-finite rows at `first` and behind it
    x = torch.ones(2, heads, dim, device="cuda").to(dtype)
    for i, at in enumerate((first, min(first + 1, m - 1))):
        k, v = x[:1].clone(), x[:1].clone()
        (k if i == 0 else v)[0, 0, 3] = math.inf if i == 0 else math.nan
        keep = [p.clone() for p in pools_of(bad)]
        one = paged.PagedBatch(torch.tensor([0, 1], device="cuda"), torch.tensor([at + 1], device="cuda"),
                               bad.table, 1, 1, None, bad.status)
        bad.cache.append(one, k, v)
        page_at, slot = bad.slots(0, at, at + 1)
        for p, q in zip(pools_of(bad), keep):  # the other heads keep their rows
            p[page_at, 1:, slot] = q[page_at, 1:, slot]
    bad.attend()
    torch.cuda.synchronize()
    assert int(bad.status) == 0
    seen = max(0, first - (m - n))
    group = q_heads // heads
    got = bad.o.double()
    assert torch.isnan(got[seen:, :group]).all()
    # a weight is rounded to 11 bits at most, from exponentials of either pipe (2^-18), the
    # output to its type: two runs differ by twice that
    most = max(float(r.abs().max()) for r in s.v)
    for a, b in ((got[:seen], sound[:seen]), (got[:, group:], sound[:, group:])):
        assert ((a - b).abs() <= (2.0 ** -10 + 2.0 ** -17) * most + 2 * U[dtype] * b.abs()).all()


def test_append_records_bad_metadata(lib, cuda):
    for change, bit in (("length", paged.BAD_LENGTH), ("offset", paged.BAD_OFFSET), ("page", paged.BAD_PAGE),
                        ("rope", paged.BAD_ROPE)):
        s = Step8([(3, 20), (0, 5), (2, 33)], 2, 2, 64, 16, F16)
        before = [p.clone() for p in pools_of(s)]
        cos, sin = s.cos, s.sin
        if change == "length":
            s.lengths[1] = 1000
        elif change == "offset":
            s.offsets[3] = 100
        elif change == "page":
            s.table[2, 1], s.table[2, 2] = -3, s.keys.shape[0]  # of tokens 31 and 32
        else:
            cos, sin = cos[:30].contiguous(), sin[:30].contiguous()
        k = torch.randn(s.tokens, 2, 64, device="cuda").half()
        s.cache.append(s.batch(), k, k, (cos, sin))
        torch.cuda.synchronize()
        assert int(s.status) == bit, change
        if change == "page":  # request 2's pages are dropped, the others' written
            where, slot = s.slots(0, 17, 20)
            after = [p.clone() for p in pools_of(s)]
            for p, a in zip(before, after):
                a[where, :, slot] = p[where, :, slot]
                assert same(p, a)


# ---- attention ------------------------------------------------------------------------------

DECODE = [(1, 1), (1, 17), (0, 40), (1, 64), (1, 129), (1, 300)]
CHUNKS = [(5, 5), (0, 0), (1, 200), (33, 97), (7, 3), (70, 130), (3, 64)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("q_heads,heads,dim,page", [(4, 4, 64, 16), (8, 2, 128, 16), (3, 1, 32, 1), (2, 2, 80, 24),
                                                    (5, 1, 256, 8), (16, 1, 16, 128), (6, 2, 48, 7), (32, 2, 64, 64),
                                                    (12, 1, 128, 8)])
@pytest.mark.parametrize("requests", [DECODE, CHUNKS], ids=["decode", "chunks"])
def test_attention_vs_float64(lib, cuda, requests, q_heads, heads, dim, page, dtype):
    s = Step8(requests, q_heads, heads, dim, page, dtype, seed=dim + page)
    s.attend()
    s.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("requests,q_heads,heads,dim", [
    ([(1, 20011)], 8, 1, 64),                          # one tile over all thread blocks
    ([(1, 5000), (1, 3), (1, 9001)], 4, 2, 128),
    ([(300, 1500)], 4, 1, 64),                         # tiles that straddle the shares
    ([(1 + b % 3, 1 + 7 * b % 130) for b in range(300)], 2, 2, 64),  # more requests than threads
    ([(257, 600), (1, 2000), (129, 129), (16, 16)], 8, 2, 128),
    ([(5, 4000), (5, 1300), (2, 2)], 8, 2, 128),       # steps of several tokens, rows in tiles of 16
    ([(300, 3000), (40, 900)], 2, 2, 256),
    ([(64, 5000)], 8, 8, 96)], ids=str)
def test_attention_divided(lib, cuda, requests, q_heads, heads, dim, dtype):
    s = Step8(requests, q_heads, heads, dim, 16, dtype, seed=len(requests))
    s.attend()
    s.check()
    first = s.o.clone()
    s.attend()
    torch.cuda.synchronize()
    assert torch.equal(first, s.o)  # the same from run to run


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("hint", [1, 3, 12, 100])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 24), (256, 16)])
def test_any_hint_is_right(lib, cuda, dim, page, hint, dtype):
    """max_new only picks the kernel."""
    s = Step8([(9, 150), (1, 260), (40, 40)], 8, 2, dim, page, dtype, seed=hint)
    s.attend(max_new=hint)
    s.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout,strided,loose", [("slots", False, False), ("heads", True, False),
                                                  ("heads", False, True), ("slots", True, True)])
@pytest.mark.parametrize("requests", [DECODE, CHUNKS], ids=["decode", "chunks"])
def test_attention_layouts(lib, cuda, requests, layout, strided, loose, dtype):
    s = Step8(requests, 8, 2, 128, 16, dtype, layout=layout, strided=strided, loose_scales=loose)
    s.attend()
    s.check()
    s.o.fill_(7.0)
    s.attend(rope=False)
    s.check(rope=False)


@pytest.mark.parametrize("q_heads,heads,dim,page", [(4, 2, 128, 16), (6, 1, 80, 8), (3, 3, 96, 64), (16, 2, 128, 128)])
@pytest.mark.parametrize("strided", [False, True])
def test_f32_chunks_above_64_dims(lib, cuda, q_heads, heads, dim, page, strided):
    """Tiles of 128 rows with sums of their own, whole and cut into parts."""
    s = Step8([(300, 2000), (130, 130), (70, 5000), (0, 7), (1, 900), (64, 3)], q_heads, heads, dim, page, F32,
              seed=dim + page, strided=strided)
    s.attend()
    s.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hint,dim", [(1, 64), (1, 128), (1, 256), (100, 64), (100, 128), (100, 256)])
def test_rows_of_any_size(lib, cuda, hint, dim, dtype):
    """Rows whose scales differ by many powers of two and rows of zeros: with up to 16 rows
    a head and where mma.sync takes the chunk, of any size; in the tcgen05 kernel (chunks up
    to 128 dims) down to 2^-21 of the largest, of the values 2^-10 here for the weights' own
    rounding of 2^-38; f32 of 128 dims there has 2^-30 here, where what is lost of such rows
    is 2^-11 of them and less than 2^-40 of the largest."""
    near = hint > 16 and dim <= (64 if dtype == F32 else 128)
    low = -10 if near else -30

    def sizes(m, heads, g):
        x = torch.exp2(torch.randint(low, 1, (m, heads, 1), device="cuda", generator=g).float())
        x[::7] = 0.0
        return x

    s = Step8([(40, 700), (20, 20), (100, 400)], 4, 2, dim, 16, dtype, seed=dim, sizes=sizes)
    s.attend(max_new=hint)
    s.check(f32_bar=2.1e-5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hint", [1, 100])
@pytest.mark.parametrize("factor", [2.0 ** -60, 2.0 ** 60])
def test_caches_of_any_size(lib, cuda, factor, hint, dtype):
    """All scales tiny or huge; the queries make up for the keys'."""
    s = Step8([(30, 300), (1, 40)], 4, 2, 64, 16, dtype, scale_factor=factor)
    s.q /= factor
    s.attend(max_new=hint)
    torch.cuda.synchronize()
    o, first = s.o.double() / factor, 0
    for b, (n, m) in enumerate(s.requests):
        q = turn(s.q[first:first + n].double(), s.cos[m - n:m], s.sin[m - n:m])
        want, _, weighted, spread = attention(q, s.k[b], s.v[b], m - n)
        delta = (2.0 ** -11 if dtype == BF16 else 2.0 ** -20) * spread
        bound = ((2 * delta).expm1() + (2.0 ** -11 if dtype == BF16 else 2e-5))[..., None] * weighted / factor
        bound = bound + U[dtype] * want.abs() / factor + 2e-5 * weighted / factor
        assert ((o[first:first + n] - want / factor).abs() <= bound).all()
        first += n


@pytest.mark.parametrize("hint", [1, 100])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_scales_that_are_no_powers_of_two(lib, cuda, hint, dtype):
    """Exact products but in the tcgen05 kernel, which rounds a row's elements to 11 bits:
    keys move scores by another 2^-11 of sum |q'||k|, values the output by 2^-11 of p|v|."""
    s = Step8([(30, 300), (2, 40)], 4, 2, 64, 16, dtype, scale_factor=1.2345)
    s.attend(max_new=hint)
    torch.cuda.synchronize()
    first = 0
    for b, (n, m) in enumerate(s.requests):
        q = turn(s.q[first:first + n].double(), s.cos[m - n:m], s.sin[m - n:m])
        o, _, weighted, spread = attention(q, s.k[b], s.v[b], m - n)
        u = 2.0 ** -11 if dtype == F16 or hint > 16 else 2.0 ** -20
        delta = 2 * u * spread + 64 * 2.0 ** -22 * spread
        bound = ((2 * delta).expm1() + 2 * u + 2e-5)[..., None] * weighted + U[dtype] * o.abs()
        assert ((s.o[first:first + n].double() - o).abs() <= bound).all()
        first += n


@pytest.mark.parametrize("hint", [1, 100])
def test_queries_of_any_size(lib, cuda, hint):
    """f16 queries at the type's ends, rows of zeros: binary16 of a scale per row.  (The
    largest of them overflow the type before the call: rows that are not finite have no
    result to compare with.)"""
    s = Step8([(24, 100)], 4, 2, 64, 16, F16, spare=0, scale_factor=2.0 ** -12)
    s.q *= torch.exp2(torch.arange(24, device="cuda").float() - 8)[:, None, None].half()
    s.q[3], s.q[4] = 0.0, 65504.0
    s.attend(max_new=hint)
    torch.cuda.synchronize()
    q = turn(s.q.double(), s.cos[76:100], s.sin[76:100])
    o, lse, weighted, spread = attention(q, s.k[0], s.v[0], 76)
    delta = 2.0 ** -11 * spread * 1.01
    bound = ((2 * delta).expm1() + 2.0 ** -11 + 2.0 ** -16)[..., None] * weighted + 2.0 ** -11 * o.abs() + 2.0 ** -25
    sound = torch.isfinite(q).all(-1)
    assert sound[:20].all()
    assert ((s.o.double() - o).abs() <= bound)[sound].all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (64, 24), (80, 7), (256, 8)])
@pytest.mark.parametrize("hint", [1, 100])
def test_bad_metadata_of_every_kernel(lib, cuda, hint, dim, page, dtype):
    """A page outside the pool reads as zeros (value 0, score 0), lengths and offsets are
    clamped, nothing outside the tensors is touched; each is recorded."""
    s = Step8([(3, 3 * page + 5), (20, 60)], 4, 2, dim, page, dtype, seed=page)
    s.table[0, 1], s.table[0, 2] = -1, s.keys.shape[0]
    for rows in (s.k, s.v):
        rows[0][page:3 * page] = 0.0
    s.attend(max_new=hint)
    s.check(status=paged.BAD_PAGE)
    s.status.zero_()
    s.lengths[1] = 1 << 40
    s.offsets[2] = s.tokens + 7
    s.o.fill_(7.0)
    s.attend(max_new=hint)
    torch.cuda.synchronize()
    assert int(s.status) & (paged.BAD_LENGTH | paged.BAD_OFFSET) == paged.BAD_LENGTH | paged.BAD_OFFSET


def test_attention_beyond_32_bits(lib, cuda):
    """Pages whose offsets in the pools (and rows whose scales') pass 2^31."""
    page, heads, dim = 64, 8, 128
    pages = (1 << 31) // (page * heads * dim) + 40
    pool = torch.zeros(2, pages, heads, page, dim, dtype=torch.uint8, device="cuda")
    scale = torch.full((2, pages, heads, page), math.nan, device="cuda")
    s = Step8([(1, 300), (40, 200)], 16, heads, dim, page, BF16)
    far = pages - 1 - torch.arange(s.table.numel(), device="cuda").reshape(s.table.shape)
    for b in range(2):
        for i, (p, sc) in enumerate(((s.keys, s.key_scales), (s.values, s.value_scales))):
            pool[i][far[b]] = p[s.table[b].long()]
            scale[i][far[b]] = sc[s.table[b].long()]
    s.cache = paged.PagedCache8(pool[0], pool[1], scale[0], scale[1], BF16)
    s.keys, s.values, s.key_scales, s.value_scales = pool[0], pool[1], scale[0], scale[1]
    s.table = far.int()
    for hint in (1, 100):
        s.attend(max_new=hint)
        s.check()
    k = torch.randn(s.tokens, heads, dim, device="cuda").bfloat16()
    s.cache.append(s.batch(), k, k, (s.cos, s.sin))
    torch.cuda.synchronize()
    where, slot = s.slots(0, 299, 300)
    bits, sc = quantise(turn_f32(k[:1], s.cos[299:300], s.sin[299:300]))
    assert torch.equal(pool[0][where, :, slot], bits) and torch.equal(scale[0][where, :, slot], sc)


@pytest.mark.parametrize("dtype,n", [(F32, 1), (BF16, 7), (F16, 90), (F32, 90)])
def test_pools_inside_one_tensor(lib, cuda, dtype, n):
    """Keys and values of all layers side by side in one tensor, as views of torch's own type:
    the same bits as in pools of their own, nothing else touched."""
    s = Step8([(n, 200), (n, n), (0, 9)], 4, 2, 64, 16, dtype)
    k, v = [torch.randn(s.tokens, 2, 64, device="cuda").to(dtype) for _ in range(2)]
    pages = s.keys.shape[0]
    every = torch.full((pages, 3, 2, 2, 16, 64), 0x11, device="cuda", dtype=torch.uint8)
    scales = torch.full((pages, 3, 2, 2, 16), 5.0, device="cuda")
    every[:, 1, 0], every[:, 1, 1], scales[:, 1, 0], scales[:, 1, 1] = pools_of(s)
    inside = paged.PagedCache8(*every.view(torch.float8_e4m3fn)[:, 1].unbind(1), *scales[:, 1].unbind(1), dtype)
    o, lse = s.o.clone(), s.lse.clone()
    rope = (s.cos, s.sin)
    inside.append(s.batch(), k, v, rope)
    paged.PagedAttention(inside, 4).forward(s.batch(), s.q, o, rope, lse)
    s.cache.append(s.batch(), k, v, rope)
    s.attend()
    torch.cuda.synchronize()
    assert int(s.status) == 0
    for a, b in zip((every[:, 1, 0], every[:, 1, 1], scales[:, 1, 0], scales[:, 1, 1]), pools_of(s)):
        assert same(a, b)
    assert torch.equal(o, s.o) and torch.equal(lse, s.lse)
    for layer in (0, 2):
        assert (every[:, layer] == 0x11).all() and (scales[:, layer] == 5.0).all()


@pytest.mark.parametrize("dtype,group,new", [(BF16, 1, 1), (F32, 4, 3), (F16, 2, 30), (F32, 2, 40)])
def test_many_requests_of_all_lengths(lib, cuda, dtype, group, new):
    """More requests than thread blocks, some without tokens, some without keys, some with more
    new tokens than they keep."""
    lengths = [(i * 37) % 131 for i in range(700)]
    requests = [(0 if i % 11 == 3 else 1 + i % new, m) for i, m in enumerate(lengths)]
    s = Step8(requests, 2 * group, 2, 32, 8, dtype)
    s.attend()
    torch.cuda.synchronize()
    assert int(s.status) == 0
    whole, lse = s.o.clone(), s.lse.clone()
    # some of them against 64 bits and against steps of their own
    first = 0
    for b, (n, m) in enumerate(requests):
        if b % 29 == 0 and n:
            at = torch.arange(m - n, m, device="cuda").clamp_min(0)
            o, want, _, _ = attention(turn(s.q[first:first + n].double(), s.cos[at], s.sin[at]), s.k[b], s.v[b], m - n)
            most = float(s.v[b].abs().max()) if m else 0.0
            assert torch.equal(torch.isinf(lse[first:first + n]), torch.isinf(want))
            assert ((whole[first:first + n].double() - o).abs() <= 2.0 ** -6 * (most + 1e-3)).all()
            one = paged.PagedBatch(torch.tensor([0, n], device="cuda"), s.lengths[b:b + 1], s.table[b:b + 1], n,
                                   new, None, s.status)
            part, part_lse = torch.empty_like(whole[first:first + n]), torch.empty_like(lse[first:first + n])
            paged.PagedAttention(s.cache, s.q_heads).forward(one, s.q[first:first + n], part, (s.cos, s.sin), part_lse)
            torch.cuda.synchronize()
            # the same products in other divisions: weights rounded to 11 bits at worst
            assert ((part.double() - whole[first:first + n].double()).abs() <=
                    2.0 ** -9 * most + 2 * U[dtype] * part.double().abs()).all()
        first += n
    assert (whole[s.used:] == 7.0).all()


def test_graphs_streams_and_workspaces(lib, cuda):
    """Captured steps follow the contents of their buffers, two graphs with their own
    workspaces replay side by side, and a workspace may hold anything."""
    made = [Step8(r, 8, 2, 128, 16, t, seed=i) for i, (r, t) in enumerate((
        ([(1, 700), (1, 90), (1, 4000)], BF16), ([(5, 600), (5, 3000)], F16), ([(200, 900)], F16),
        ([(70, 500)], F32)))]
    objects = [paged.PagedAttention(s.cache, 8) for s in made]
    streams = [torch.cuda.Stream() for _ in made]
    graphs, first = [], []
    for s, a, stream in zip(made, objects, streams):
        a.ws.fill_(255)
        b = s.batch()
        s.attend(attention_object=a)
        s.check()
        first.append(s.o.clone())
        a.ws.fill_(255)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            a.forward(b, s.q, s.o, (s.cos, s.sin), s.lse)
        graphs.append(graph)
        s.o.fill_(7.0)
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for s, o in zip(made, first):
        assert torch.equal(s.o, o)
    s = made[0]
    s.lengths.copy_(torch.tensor([650, 1, 3999], device="cuda"))
    s.requests = [(1, 650), (1, 1), (1, 3999)]
    for b, (_, m) in enumerate(s.requests):
        s.k[b], s.v[b] = s.k[b][:m], s.v[b][:m]
    torch.cuda.synchronize()
    graphs[0].replay()
    s.check()


def test_calls_from_several_threads(lib, cuda):
    """Host threads with streams and workspaces of their own, kernels of every kind at once."""
    made = [Step8(r, 8, 2, d, p, t, seed=i) for i, (r, d, p, t) in enumerate((
        ([(1, 3000)] * 5, 128, 16, BF16), ([(6, 500), (40, 40)], 64, 24, F16), ([(90, 700)], 128, 64, F32),
        ([(200, 300), (3, 900)], 128, 16, BF16)))]
    for s in made:
        s.attend()
    torch.cuda.synchronize()
    alone = [(s.o.clone(), s.lse.clone()) for s in made]
    for s in made:
        s.o.zero_(), s.lse.zero_()
    torch.cuda.synchronize()
    failed = []

    def work(s):
        try:
            stream = torch.cuda.Stream()
            attention_object = paged.PagedAttention(s.cache, s.q_heads)
            for _ in range(20):
                s.attend(stream=stream.cuda_stream, attention_object=attention_object)
            stream.synchronize()
        except Exception as e:  # reported by the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in made]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for s, (o, lse) in zip(made, alone):
        rows = slice(0, s.used)
        assert torch.equal(s.o[rows], o[rows]) and torch.equal(s.lse[rows], lse[rows]) and int(s.status) == 0


def test_calls_follow_the_current_stream(lib, cuda):
    """Without a stream of its own a call runs behind what torch's current one holds."""
    s = Step8([(4, 200), (1, 900)], 4, 2, 64, 16, F16)
    s.attend()
    s.check()
    want, q = s.o.clone(), s.q.clone()
    side = torch.cuda.Stream()
    s.q.zero_()
    s.o.fill_(7.0)
    a = paged.PagedAttention(s.cache, 4)
    b = s.batch()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        s.q.copy_(q)
        a.forward(b, s.q, s.o, (s.cos, s.sin), s.lse)
    side.synchronize()
    assert torch.equal(s.o, want)


def test_python_refusals(lib, cuda):
    s = Step8([(1, 20)], 2, 1, 64, 16, F16, spare=0)
    ok = (s.keys, s.values, s.key_scales, s.value_scales)
    for bad in ((s.keys.cpu(),) + ok[1:], (s.keys, s.values[:1]) + ok[2:], (s.keys.int(), s.values.int()) + ok[2:],
                ok[:2] + (s.key_scales[:1], s.value_scales), ok[:3] + (s.value_scales.double(),),
                ok[:2] + (s.key_scales, s.value_scales.transpose(0, 2).contiguous().transpose(0, 2)),
                (s.keys[..., ::2], s.values[..., ::2]) + ok[2:]):
        with pytest.raises(ValueError):
            paged.PagedCache8(*bad, F16)
    with pytest.raises(ValueError):
        paged.PagedCache8(*ok, torch.float64)
    for a in (paged.PagedCache8(s.keys.view(torch.float8_e4m3fn), s.values.view(torch.float8_e4m3fn), *ok[2:], F16),):
        o = s.o.clone()
        paged.PagedAttention(a, 2).forward(s.batch(), s.q, o)
    with pytest.raises(ValueError):
        paged.PagedAttention(s.cache, 2).forward(s.batch(), s.q.float(), s.o)
    with pytest.raises(ValueError):
        s.cache.append(s.batch(), s.q.float()[:, :1], s.q[:, :1])
    with pytest.raises(ValueError):
        paged.PagedAttention(s.cache, 0)
    with pytest.raises(Exception):
        narrow = torch.zeros(4, 1, 16, 24, dtype=torch.uint8, device="cuda")  # 24 dims
        sc = torch.zeros(4, 1, 16, device="cuda")
        k = torch.zeros(1, 1, 24, dtype=F16, device="cuda")
        paged.PagedCache8(narrow, narrow, sc, sc, F16).append(s.batch(), k, k)
