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
import sys
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
