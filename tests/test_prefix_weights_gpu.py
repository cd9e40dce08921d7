"""Weights of the attention of a shared prefix at the ends of their range (needs a B200)."""
import numpy as np
import pytest
import torch

import serve_ref as R
from serve_ref import DEV, DT, HALF
from test_prefix_gpu import Batch

pytestmark = pytest.mark.gpu

# (tokens, query heads, KV heads, head size, prefix, own slots): row tiles whose whole prefix one CTA reads, prefixes cut into parts, prefixes that the
# blocks of the own slots read, own slots alone and beside a prefix, heads that share a block's rows
SHAPES = [(600, 64, 8, 64, 20000, 1), (300, 64, 8, 128, 20000, 20), (33, 32, 8, 128, 9000, 30), (3, 8, 8, 64, 3000, 7000), (1, 32, 8, 128, 600, 1), (1, 16, 1, 64, 0, 8000), (40, 12, 4, 128, 0, 3000)]


def only(b, tokens):
    """The batch's outputs of a few tokens, for a check."""
    b.o, b.q, b.tok_seq, b.ctx, b.n = b.o[tokens], b.q[tokens], b.tok_seq[tokens], b.ctx[tokens], len(tokens)


@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("tokens,nh,nkvh,dh,prefix,own", SHAPES)
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -5, 2.0 ** -8, 2.0 ** -20])
def test_scores_of_billions(L, dt, tokens, nh, nkvh, dh, prefix, own, scale):
    """Scores are single products, exact in 32 bits, up to 2.8e9 times the scale.  Several keys have the largest, so their weights are one, however large
    that is, and all others' are zero (the next score is 384 below at the smallest scale).  Sums of weights are whole multiples of one below 2^24; sums of
    values take a rounding for every 16 positions (2^-23: truncation counts double), 64 for parts and quotients, and the result is rounded."""
    b = Batch(tokens + prefix, [(own, 1)] * tokens, prefix, nh, nkvh, dh, dt, 64)
    b.pool[:, 0] = 0.0
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    pick = torch.randint(0, 40, b.pool[:, 0, ..., 0].shape, generator=g, device=DEV)
    b.pool[:, 0, ..., 7] = torch.where(pick == 0, 57344.0, torch.where(pick < 20, 49152.0, -57344.0)).to(DT[dt])
    first = int((b.prefix_ids if prefix else b.ids[0])[0])
    b.pool[first, 0, :, 0, 7] = 57344.0  # everyone sees one of the largest
    if not prefix:
        b.ids[:, 0] = first
    b.q.zero_()
    b.q[..., 7] = 49152.0
    b.scale = scale
    b.run(L)
    only(b, list(range(0, tokens, 97)))
    shared = b.rows(b.prefix_ids, b.prefix)
    for t in range(b.n):
        mine = b.rows(b.ids[b.tok_seq[t]], int(b.ctx[t]))
        want, mag = R.attention(b.q[t], *shared, *mine, scale)
        off = (b.o[t].double() - want).abs()
        tol = HALF[dt] * want.abs() + ((prefix + own) / 16 + 64) * 2.0 ** -23 * mag + 2.0 ** -24
        assert b.o[t].isfinite().all() and (off <= tol).all(), f"token {t}: {float(off.max())} off, {float((off / tol).max())} of what is allowed"


@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("tokens,nh,nkvh,dh,prefix,own", SHAPES)
@pytest.mark.parametrize("below", [25.1, 27.5])
def test_many_keys_far_below_one(L, dt, tokens, nh, nkvh, dh, prefix, own, below):
    """The first key of all outweighs each of the others 2^25.1 and 2^27.5 times, but these are thousands, and their values are all the result there
    is.  A weight may be off by half a step of its type, as in any batch."""
    page = 64
    b = Batch(tokens + prefix, [(own, 1)] * tokens, prefix, nh, nkvh, dh, dt, page)
    sink, flat = (int(p) for p in (b.prefix_ids if prefix else b.ids[0])[:2])
    b.prefix_ids[1:] = flat
    b.ids[:] = flat
    if not prefix:
        b.ids[:, 0] = sink
    b.pool.zero_()
    b.pool[:, 1] = 512.0
    b.pool[sink, 1, :, 0] = 0.0
    b.q.zero_()
    b.q[..., 5] = 8.0
    b.scale = 0.125
    b.pool[sink, 0, :, 0, 5] = below * float(np.log(2.0))  # (rounded to the type: the check reads what is there)
    b.run(L)
    only(b, list(range(0, tokens, 97)))
    b.check()
