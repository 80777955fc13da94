"""The 8-bit paged cache where its pages, scales and rows are unusual."""
import pytest
import torch

from test_gpu_cache8 import BF16, F16, F32, Step8
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
