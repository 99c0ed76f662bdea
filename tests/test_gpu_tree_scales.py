"""Tree attention over coded caches whose rows' scales lie far apart: a row weighs what its own scale says, whatever the
scales of the rows beside it are, attended or not."""
import math

import numpy as np
import pytest

import treeref
from test_gpu_tree import Case

pytestmark = pytest.mark.gpu

CODED = ["int8", "fp8", "int4", "fp4"]


def attend(q, k, v, ks, vs, kv):
    """Attention of q over all of k and v in 64 bits, and how far a float evaluation with weights in two bf16 halves may be
    from it.

    Scores as in treeref.attend: 74 roundings of 2^-24 of the sum of magnitudes (INT4 codes count 15 + 8), twice, since
    the maximum has them too.  A weight is exp2 of that (2^-22), its product with its row's scale rounds once, and the
    product is cut to two halves: the upper cut leaves less than 2^-7 of it, the cut of the rest less than 2^-7 of that.
    Sums: of each 32 rows of a product, the joins and the division, a rounding of what the rows have added up to: of every
    row's own weight times its largest code (INT4: 23) times its scale.  Then half a step of the output."""
    s = k @ q / 8.0
    w = np.exp(s - s.max())
    w /= w.sum()
    ref = w @ v
    more = 23.0 if kv == "int4" else 0.0
    mag = (np.abs(k) @ np.abs(q) + more * np.abs(q).sum() * ks * (more > 0)).max()
    es = 2 * 74 * 2.0 ** -24 * mag * 0.125 * math.log2(math.e)
    rel_w = 2.0 ** -14 + 2.0 ** -21 + 2 * math.log(2) * es
    largest = {"int8": 127.0, "fp8": 448.0, "int4": 23.0, "fp4": 6.0}[kv]
    steps = (len(k) / 32 + 24) * 2.0 ** -24
    return ref, 2.0 ** -8 * np.abs(ref) + 2 * rel_w * (w @ np.abs(v)) + 2 * steps * largest * (w @ vs) + 2.0 ** -126


def check(c, got):
    for b in range(c.B):
        for h in range(c.NH):
            k, v, ks, vs, ok = c.rows(b, h)
            for i in range(c.sizes[b]):
                t = c.start[b] + i
                seen = c.seen(b, i)
                seen = seen[ok[seen]]
                ref, bound = attend(c.q[t, 0, h].astype(np.float64), k[seen], v[seen], ks[seen], vs[seen], c.kv)
                err = np.abs(got[t, h] - ref)
                assert (err <= bound).all(), (b, h, i, float((err / bound).max()))


def _row(c, b, i):
    pos = c.lens[b] - c.sizes[b] + i
    return c.table[b][pos // c.R], pos % c.R


@pytest.mark.parametrize("kv", CODED)
@pytest.mark.parametrize("sizes,lens,S", [([26, 9], [300, 130], 0), ([40, 1], [700, 64], 3), ([16], [16], 0)])
def test_ordinary_scales(dev, kv, sizes, lens, S):
    c = Case(dev, kv, sizes, lens, 2, 64, seed=71)
    check(c, c.run(S=S))


@pytest.mark.parametrize("kv", CODED)
@pytest.mark.parametrize("scale", [1e7, 1e20, 1e30])
def test_large_scales_of_rows_that_are_not_attended(dev, kv, scale):
    """A branch's V rows with large scales beside another's; who attends one has it."""
    c = Case(dev, kv, [40, 20], [200, 20], 2, 64, seed=72)
    for b, i in ((0, 3), (0, 22), (1, 6)):
        page, row = _row(c, b, i)
        c.scale[page, 1, :, row] = scale
    others = [t for b, i in ((0, 3), (1, 6)) for t in range(c.start[b], c.start[b + 1]) if not (int(c.masks[t, 0]) >> i) & 1]
    assert others
    check(c, c.run())
    # K's alone: a score that is not looked at.
    c = Case(dev, kv, [40, 20], [200, 20], 2, 64, seed=72)
    page, row = _row(c, 0, 39)
    c.scale[page, 0, :, row] = scale
    c.masks[c.start[0] + 39, 0] &= ~np.uint64(1 << 39)
    check(c, c.run())


@pytest.mark.parametrize("kv", CODED)
@pytest.mark.parametrize("scale", [1e7, 1e30])
@pytest.mark.parametrize("missing", [[(0, 0)], [(0, 1), (0, 2)], [(0, 0), (0, 9), (1, 0)]])
def test_large_scales_beside_missing_pages(dev, kv, scale, missing):
    """The pool's first page, in no table, and pages that stand before a missing one."""
    c = Case(dev, kv, [18, 5], [640, 128], 2, 64, seed=73, missing=missing)
    c.table[c.table == 0] = int(np.setdiff1d(np.arange(c.P), c.table)[0])
    c.scale[0] = scale
    check(c, c.run())
    check(c, c.run(S=2))


@pytest.mark.parametrize("kv", CODED)
@pytest.mark.parametrize("spread", [12, 40])
def test_scales_far_apart(dev, kv, spread):
    """Attended rows of a tile with scales far apart: small ones with most of the weight count beside large ones with next
    to none."""
    c = Case(dev, kv, [18, 6], [500, 130], 2, 64, seed=74, sharp=3.0)
    r = np.random.RandomState(75)
    import torch
    f = np.exp2(r.randint(-spread, spread + 1, c.scale[:, 1].shape).astype(np.float32))
    c.scale[:, 1] *= torch.from_numpy(f)
    check(c, c.run())
    check(c, c.run(S=4))


@pytest.mark.parametrize("kv", CODED)
def test_rows_that_weigh_nothing(dev, kv):
    """One row has a large V scale and a score so low that it adds nothing: the others' outputs stay."""
    c = Case(dev, kv, [4], [200], 1, 64, seed=76)
    page, row = c.table[0][70 // c.R], 70 % c.R
    c.scale[page, 1, 0, row] = 1e9
    c.stored[page, 0, 0, row] = {"int8": 127, "fp8": 0x7E, "int4": 0xFF, "fp4": 0x77}[kv]      # K: the largest code
    c.scale[page, 0, 0, row] = 1.0
    c.q[:, 0] = -np.abs(c.q[:, 0]) - 8.0
    c.q = treeref.bf16(c.q)
    got = c.run()
    assert np.abs(got).max() < 8.0
    check(c, got)
