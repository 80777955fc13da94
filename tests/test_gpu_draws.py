"""The draw of et_b200_verify_v1 over many segments of the vocabulary, in clusters of every size:
tokens far apart, on both sides of every border, the second attempt, rows without mass.

Probabilities are whole multiples of 2^-12 on a few dozen tokens, so every sum is exact in
whatever order, and draws aim at the middle of a token: every id is known.
"""
import numpy as np
import pytest
import torch

from eshkol_transformer_b200 import sampling

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -12
KINDS = 6


def tokens_of(vocab, rng):
    """Tokens in order: the ends, both sides of segments' borders, any others."""
    at = {0, vocab - 1, 1023, 1024, (vocab - 1) // 1024 * 1024, (vocab - 1) // 1024 * 1024 - 1}
    while len(at) < 40:
        at.add(int(rng.integers(vocab)))
    return np.array(sorted(at))


def drawn(tokens, weights, u):
    """The first token whose running sum exceeds u times the total (1 and more: the last that
    weighs something)."""
    run = np.cumsum(weights)
    if run[-1] == 0:
        return -1
    some = np.nonzero(weights)[0]
    over = [i for i in some if run[i] > u * run[-1]]
    return int(tokens[over[0] if over else some[-1]])


def middle(weights, i):
    return (np.cumsum(weights)[i] - 0.5 * weights[i]) / weights.sum()


class Requests:
    """Requests of six kinds in turn, two rows each: a proposal that is accepted; one that is not,
    with a rest of p - q; p <= q everywhere; no mass; a draw at 1; no rest and a draw at 1."""

    def __init__(self, vocab, batch, chance, seed=1):
        rng = np.random.default_rng(seed)
        self.tokens = tokens_of(vocab, rng)
        count, rows = len(self.tokens), 2 * batch
        p, q = np.zeros((rows, count), np.int64), np.zeros((rows, count), np.int64)
        drafts, accept = np.zeros(rows, np.int64), np.zeros(rows)
        draw = np.zeros(batch)
        ids, accepted = np.full(rows, -1, np.int64), np.zeros(batch, np.int64)
        for b in range(batch):
            r, kind = 2 * b, b % KINDS
            for i in (r, r + 1):
                p[i] = rng.integers(1, 30, count)
                p[i, 0 if i % 4 < 2 else -1] = 200
            target, goal = r, (b * 17 + b // KINDS) % count
            x = int(rng.integers(count))
            if kind == 0:
                q[r, x], accept[r], target = 5, 0.0, r + 1
                rest = p[target]
                ids[r], accepted[b] = self.tokens[x], 1
            else:
                q[r] = rng.integers(0, 30, count)
                p[r, x], q[r, x], accept[r] = 0, 7, 0.5
                if kind in (2, 5):
                    q[r] = np.maximum(p[r], q[r])
                if kind == 3:
                    p[r] = 0
                if not chance:  # q is 1 at the proposal: the rest is p without it
                    q[r] = 0
                rest = np.maximum(p[r] - q[r], 0)
                if rest.sum() == 0:
                    rest = p[r]
            drafts[r] = self.tokens[x]
            drafts[r + 1] = 1 << 60  # not read
            if kind in (4, 5):
                draw[b] = 1.0
            elif rest.sum() > 0:
                some = np.nonzero(rest)[0]
                draw[b] = middle(rest, some[goal % len(some)])
            ids[target] = drawn(self.tokens, rest, draw[b])
        dev = lambda a, t: torch.as_tensor(a, dtype=t, device="cuda")
        where = dev(self.tokens, torch.int64)

        def spread(a):
            t = torch.zeros(rows, vocab, device="cuda")
            t[:, where] = dev(a * UNIT, torch.float32)
            return t

        self.target, self.draft = spread(p), spread(q) if chance else None
        self.drafts, self.accept = dev(drafts, torch.int64), dev(accept, torch.float32)
        self.draw = dev(draw, torch.float32)
        self.offsets = torch.arange(batch + 1, device="cuda") * 2
        self.want_ids, self.want_accepted = ids, accepted
        self.verifier = sampling.Verifier(batch, rows, vocab)

    def run(self):
        ids, accepted = torch.full_like(self.drafts, -9), torch.full_like(self.offsets[:-1], -9)
        self.verifier.verify(self.offsets, self.target, self.drafts, self.draft, self.accept, self.draw, ids,
                             accepted)
        return ids.cpu().numpy(), accepted.cpu().numpy()


# up to 37 requests take clusters of 8 thread blocks, up to 74 of 4, up to 148 of 2, more of one
@pytest.mark.parametrize("chance", [True, False])
@pytest.mark.parametrize("vocab,batch", [
    (128259, 1), (128259, 30), (128259, 60), (128259, 90), (128259, 160), (524288, 30), (524289, 1),
    (524289, 30), (600001, 1), (600001, 30), (600001, 60), (600001, 90), (600001, 160), (1 << 22, 1),
    (1 << 22, 30), (1 << 22, 80)])
def test_every_draw_is_the_one_asked_for(lib, cuda, vocab, batch, chance):
    for seed in range(KINDS if batch == 1 else 1):  # a single request is of each kind in turn
        r = Requests(vocab, batch, chance, seed)
        if batch == 1 and seed:
            other = Requests(vocab, KINDS, chance, seed)
            rows = slice(2 * seed, 2 * seed + 2)
            r.target = other.target[rows].contiguous()
            r.draft = None if other.draft is None else other.draft[rows].contiguous()
            r.drafts, r.accept, r.draw = other.drafts[rows], other.accept[rows], other.draw[seed:seed + 1]
            r.want_ids, r.want_accepted = other.want_ids[rows], other.want_accepted[seed:seed + 1]
        for _ in range(5):
            ids, accepted = r.run()
            assert (accepted == r.want_accepted).all()
            assert (ids == r.want_ids).all(), np.nonzero(ids != r.want_ids)
