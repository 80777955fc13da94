"""The 8-bit paged cache where its pages, scales and rows are unusual."""
import pytest
import torch

from cache8_f64 import rows_of
from test_gpu_cache8 import BF16, F16, F32, Step8, appended, pools_of, same
from eshkol_transformer_b200 import paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 8), (128, 64), (256, 16), (80, 24)])
@pytest.mark.parametrize("hint", [1, 4, 20, 100])
def test_bad_pages_among_sound_ones(lib, cuda, hint, dim, page, dtype):
    """Pages outside the pool among sound ones, so that every stage's scales are zeros by plain stores
    and copies in turn: the bits of a cache that holds a page of zeros there."""
    s = Step8([(5, 3000), (1, 1500), (33, 2000)], 4, 2, dim, page, dtype, seed=dim + hint)
    g = torch.Generator(device="cuda").manual_seed(hint)
    bad = torch.rand(s.table.shape, device="cuda", generator=g) < 0.4
    free = torch.ones(s.keys.shape[0], dtype=torch.bool, device="cuda")
    free[s.table.flatten().long()] = False
    zeros = int(free.nonzero()[0])  # a page that no request has
    for pool in (s.keys, s.values, s.key_scales, s.value_scales):
        pool[zeros] = 0
    table = s.table.clone()
    s.table = torch.where(bad, zeros, table)
    s.attend(max_new=hint)
    torch.cuda.synchronize()
    assert int(s.status) == 0
    want, lse = s.o.clone(), s.lse.clone()
    outside = torch.where(torch.rand(table.shape, device="cuda", generator=g) < 0.5, -1, s.keys.shape[0])
    s.table = torch.where(bad, outside.int(), table)
    for _ in range(3):
        s.o.fill_(7.0), s.lse.fill_(7.0), s.status.zero_()
        s.attend(max_new=hint)
        torch.cuda.synchronize()
        assert int(s.status) == paged.BAD_PAGE
        assert torch.equal(s.o, want) and torch.equal(s.lse, lse)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("hint", [1, 4, 100])
def test_small_rows_beside_large_ones(lib, cuda, hint, dim, dtype):
    """Rows of keys and of values whose scales are 2^-21 of the largest of their block keep every
    bit, in every kernel: the large keys lie where no query looks (their scores are below -1,000), so
    the outputs are means of the small values alone.

    With u = 2^-11 (f32: 2^-22) for queries and weights, a score of a small key is off by delta =
    (u + dim 2^-23 + 2^-22) sum |q||k|, its weight by exp(2 delta) - 1 and by u relative and by 2^-36 of
    the largest, sums over m keys by (m + 16) 2^-23 and exponentials by 2^-17 where the type is of 16
    bits, by 2e-5 at f32; the output by half a step."""
    s = Step8([(100, 700), (64, 300), (70, 170)], 4, 2, dim, 16, dtype, seed=dim)
    g = torch.Generator(device="cuda").manual_seed(dim + hint)
    s.q.copy_(torch.randn(s.q.shape, device="cuda", generator=g) * 2.0 ** 8)
    s.q[..., 0] = (s.q[..., 0].abs() + 2.0 ** 8).to(dtype)
    u, step = (2.0 ** -22, 2.0 ** -24) if dtype == F32 else (2.0 ** -11, 2.0 ** (-11 if dtype == F16 else -8))
    large = []
    for b, (_, m) in enumerate(s.requests):
        where, slot = s.slots(b, 0, m)
        large.append(torch.rand(m, 2, device="cuda", generator=g) < 0.3)
        bits = s.keys[where, :, slot]
        bits[large[b]] = 0
        bits[..., 0] = torch.where(large[b], 0xc8, bits[..., 0].int()).byte()  # -4
        s.keys[where, :, slot] = bits
        s.key_scales[where, :, slot] = torch.where(large[b], 2.0 ** 5, 2.0 ** -16)
        s.value_scales[where, :, slot] = torch.where(large[b], 2.0 ** 6, 2.0 ** -15)
        s.k[b] = rows_of(s.keys[where, :, slot], s.key_scales[where, :, slot])
        s.v[b] = rows_of(s.values[where, :, slot], s.value_scales[where, :, slot])
    s.attend(rope=False, max_new=hint)
    torch.cuda.synchronize()
    assert int(s.status) == 0
    first = 0
    for b, (n, m) in enumerate(s.requests):
        q, got = s.q[first:first + n].double(), s.o[first:first + n].double()
        lse = s.lse[first:first + n].double()
        first += n
        hidden = torch.arange(m, device="cuda") > torch.arange(m - n, m, device="cuda")[:, None]
        for h in range(4):
            k, v, far = s.k[b][:, h // 2], s.v[b][:, h // 2], large[b][:, h // 2]
            x = (q[:, h] @ k.T / dim ** 0.5).masked_fill(hidden, -torch.inf)
            assert (x[:, far] < -1000).all() and x[:, ~far].abs().nan_to_num(posinf=0.0).amax() < 256
            p, small = torch.softmax(x, 1)[:, ~far], v[~far]
            want, weighted = p @ small, p @ small.abs()
            spread = (q[:, h].abs() @ k[~far].abs().T / dim ** 0.5).amax(1, keepdim=True)
            delta = (u + dim * 2.0 ** -23 + 2.0 ** -22) * spread
            sums = 2e-5 if dtype == F32 else (m + 16) * 2.0 ** -23 + 2.0 ** -17
            bound = ((2 * delta).expm1() + u + sums) * weighted + m * 2.0 ** -36 * small.abs().max()
            bound = bound + step * want.abs() + (2.0 ** -25 if dtype == F16 else 0.0)
            assert ((got[:, h] - want).abs() <= bound).all()
            room = delta[:, 0] + 2e-5 * (1 + torch.logsumexp(x, 1).abs())
            assert ((lse[:, h] - torch.logsumexp(x, 1)).abs() <= room).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_append_leaves_zeros_under_scales_that_are_nan(lib, cuda, dtype):
    """Every byte of the pools, those of rows that are not finite included: zeros, which a query that does
    not see them multiplies by 0."""
    s = Step8([(40, 40), (3, 50)], 2, 2, 64, 16, dtype)
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(s.tokens, 2, 64, device="cuda", generator=g).to(dtype) for _ in range(2))
    for x in (k, v):
        for i, bad in enumerate((torch.inf, -torch.inf, torch.nan)):
            x[5 + 4 * i, i % 2, 7 * i] = bad
            x[41, i % 2, 63] = bad
    for rope in (True, False):
        want = appended(s, k, v, rope)
        s.cache.append(s.batch(), k, v, (s.cos, s.sin) if rope else None)
        torch.cuda.synchronize()
        assert int(s.status) == 0
        for got, w in zip(pools_of(s), want):
            assert same(got, w)
        where, slot = s.slots(0, 0, 40)
        none = torch.isnan(s.value_scales[where, :, slot])
        assert int(none.sum()) == 3 and (s.values[where, :, slot][none] == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("group,dim,page,new", [(4, 32, 8, 3), (2, 32, 8, 40), (4, 64, 16, 9), (1, 128, 24, 5),
                                                (8, 128, 16, 12)])
def test_hundreds_of_requests_against_float64(lib, cuda, group, dim, page, new, dtype):
    """More requests than thread blocks, some without tokens, some without keys, some with more new tokens
    than they keep; every one of them by the bounds of the few."""
    requests = [(0 if i % 11 == 3 else 1 + i % new, (i * 37) % 131) for i in range(400)]
    s = Step8(requests, 2 * group, 2, dim, page, dtype, seed=new)
    s.attend()
    s.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,page", [(256, 16), (128, 24), (112, 7), (64, 24)])
@pytest.mark.parametrize("new", [5, 12, 13, 48, 49])
def test_rows_around_the_kernels_borders(lib, cuda, new, dim, page, dtype):
    """20 to 196 rows per kv head where no tcgen05 kernel takes the cache."""
    s = Step8([(new, 900), (new // 2, 40), (1, 2000), (new, new)], 8, 2, dim, page, dtype, seed=new)
    s.attend()
    s.check()
    first = s.o.clone()
    s.attend()
    torch.cuda.synchronize()
    assert torch.equal(first, s.o)
