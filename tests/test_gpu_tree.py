"""Trees of drafted tokens: masks from parents, attention over paged caches of every type, and the accepted paths' rows,
against restatements in 64 bits (treeref)."""
import numpy as np
import pytest

import treeref
from treeref import HS

pytestmark = pytest.mark.gpu

KINDS = ["f32", "bf16", "int8", "fp8", "int4", "fp4"]


def _kv():
    from cuda_gpt2_inference_amd import kvattn
    return kvattn


def _dev(x, dev, dtype=None):
    import torch
    x = np.ascontiguousarray(x)
    t = torch.from_numpy(x.view(np.int64) if x.dtype == np.uint64 else x).to(dev)
    return t if dtype is None else t.to(dtype)


@pytest.mark.parametrize("words,sizes", [(1, [1, 0, 5, 64, 2]), (2, [100, 128, 65, 1]), (4, [256, 0, 0, 193]), (1, [70, 3]),
                                         (4, [300, 7]), (3, [130])])
def test_masks(dev, words, sizes):
    import torch
    r = np.random.RandomState(len(sizes) * 10 + words)
    start, parents = treeref.forest(r, sizes, wild=True)
    lens = r.randint(0, 2000, len(sizes)).astype(np.int32)
    N = len(parents)
    got = torch.full((N + 2, words), -5, dtype=torch.int64, device=dev)
    pos = torch.full((N + 2,), -5, dtype=torch.int32, device=dev)
    _kv().tree_masks(got, _dev(parents, dev), _dev(start, dev), len(sizes), N + 2, positions=pos, lens=_dev(lens, dev),
                     mask_words=words)
    want, depth = treeref.masks(start, parents, words)
    assert np.array_equal(got.cpu().numpy().view(np.uint64)[:N], want) and (got[N:] == -5).all()
    n = np.repeat(np.diff(start), np.diff(start))
    assert np.array_equal(pos.cpu().numpy()[:N], np.maximum(np.repeat(lens, sizes) - n + depth, 0)) and (pos[N:] == -5).all()
    again = torch.zeros_like(got)
    _kv().tree_masks(again, _dev(parents, dev), _dev(start, dev), len(sizes), N, mask_words=words)
    assert torch.equal(again[:N], got[:N])


class Case:
    """A pool, its tables and a forest on the device, and the reference's view of them."""

    def __init__(self, dev, kv, sizes, lens, NH, R, words=1, seed=0, sharp=1.0, missing=()):
        import torch
        r = np.random.RandomState(seed)
        self.kv, self.NH, self.R, self.sizes, self.lens, self.words = kv, NH, R, sizes, lens, words
        self.B = len(sizes)
        self.start, self.parents = treeref.forest(r, sizes)
        self.N = len(self.parents)
        self.max_pages = max(1, -(-max(max(lens), 1) // R))
        P = self.B * self.max_pages + 1
        self.x = r.standard_normal((P, 2, NH, R, HS)).astype(np.float32)
        if kv == "bf16":
            self.x = treeref.bf16(self.x)
        self.stored, self.scale = treeref.encode(self.x, kv)
        self.table = r.permutation(P)[:self.B * self.max_pages].reshape(self.B, self.max_pages).astype(np.int32)
        for b, i in missing:
            self.table[b, i] = P + 3 if (b + i) % 2 else -1
        self.P = P
        q = (sharp * r.standard_normal((self.N, 3, NH, HS))).astype(np.float32)
        self.q = q if kv == "f32" else treeref.bf16(q)
        self.masks, _ = treeref.masks(self.start, self.parents, words)
        self.dev = dev
        self.act = torch.float32 if kv == "f32" else torch.bfloat16

    def run(self, S=0, max_new=None, spare=3):
        import torch
        kvattn = _kv()
        rows = self.N + spare
        qkv = torch.zeros((rows, 3, self.NH, HS), dtype=self.act, device=self.dev)
        qkv[:self.N] = torch.from_numpy(self.q).to(self.act).to(self.dev)
        masks = torch.zeros((rows, self.words), dtype=torch.int64, device=self.dev)
        masks[:self.N] = _dev(self.masks, self.dev)
        out = torch.full((rows, self.NH, HS), 77.0, dtype=self.act, device=self.dev)
        cache = kvattn.PagedCache(self.stored.to(self.dev), _dev(self.table, self.dev), self.max_pages, self.R, self.P,
                                  None if self.scale is None else self.scale.to(self.dev))
        ws = kvattn.Workspace(rows, self.NH, self.max_pages * self.R, S=S)
        before = ws.buf.clone()
        args = (out, qkv, cache, _dev(self.start, self.dev), _dev(np.array(self.lens, dtype=np.int32), self.dev), masks, self.B,
                rows, self.NH, HS)
        kw = dict(kv_dtype=self.kv, max_new=max_new or max(max(self.sizes), 1), mask_words=self.words, S=S, **ws.kwargs())
        kvattn.paged_decode_tree(*args, **kw)
        first = out.clone()
        kvattn.paged_decode_tree(*args, **kw)                    # the counters are as they were
        torch.cuda.synchronize()
        assert torch.equal(first.view(torch.uint8), out.view(torch.uint8))
        assert torch.equal(ws.buf[:256], before[:256])
        assert (out[self.N:] == 77.0).all()
        return out[:self.N].double().cpu().numpy()

    def rows(self, b, h):
        """K, V [total][HS], their scales, and which positions are there."""
        T = self.lens[b]
        page = self.table[b][np.arange(T) // self.R]
        ok = (page >= 0) & (page < self.P)
        page, row = np.where(ok, page, 0), np.arange(T) % self.R
        out = []
        for part in (0, 1):
            sc = None if self.scale is None else self.scale[page, part, h, row]
            out.append(treeref.decode(self.stored[page, part, h, row], sc, self.kv))
            out.append(None if sc is None else sc.numpy().astype(np.float64))
        return out[0], out[2], out[1], out[3], ok

    def seen(self, b, i):
        """Positions that token i of sequence b attends."""
        T, n, t0 = self.lens[b], self.sizes[b], self.start[b]
        base = T - n
        s = list(range(max(0, base)))
        for j in range(min(n, 64 * self.words)):
            if (int(self.masks[t0 + i, j >> 6]) >> (j & 63)) & 1 and base + j >= 0:
                s.append(base + j)
        return np.array(s, dtype=np.int64)

    def check(self, got, tokens=None):
        worst = 0.0
        for b in range(self.B):
            for h in range(self.NH):
                if self.sizes[b] == 0:
                    continue
                k, v, ks, vs, ok = self.rows(b, h)
                for i in range(self.sizes[b]):
                    t = self.start[b] + i
                    if tokens is not None and i >= tokens:
                        continue
                    seen = self.seen(b, i)
                    seen = seen[ok[seen]] if len(seen) else seen
                    with np.errstate(invalid="ignore", over="ignore"):
                        ref, bound = treeref.attend(self.q[t, 0, h].astype(np.float64), k, v, seen, ks, vs, self.kv)
                    err = np.abs(got[t, h] - ref)
                    assert (err <= bound).all(), (self.kv, b, h, i, float((err / bound).max()))
                    worst = max(worst, float((err / bound).max()))
        return worst


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("sizes,lens,NH,R,S", [
    ([1], [1], 1, 64, 0),                                # one token alone
    ([5], [5], 2, 64, 0),                                # no prefix
    ([16, 3, 0, 17], [64, 65, 100, 130], 3, 64, 0),      # tiles' ends, a sequence without tokens
    ([33, 64, 1], [200, 64, 190], 2, 192, 0),
    ([26], [700], 2, 128, 0),                            # segments
    ([7, 40], [900, 333], 2, 64, 3),
    ([7, 40], [900, 333], 2, 64, -64),
    ([12], [1000], 1, 64, 1),
])
def test_attention(dev, kv, sizes, lens, NH, R, S):
    c = Case(dev, kv, sizes, lens, NH, R, seed=len(sizes) + lens[0])
    c.check(c.run(S=S))


@pytest.mark.parametrize("kv", KINDS)
def test_attention_large_trees(dev, kv):
    """More tokens than a workgroup holds; masks of several words; new tokens over several tiles."""
    c = Case(dev, kv, [150, 0, 70, 256], [300, 50, 70, 600], 1, 64, words=4, seed=5)
    c.check(c.run())
    c = Case(dev, kv, [65, 128], [129, 500], 1, 128, words=2, seed=6)
    c.check(c.run(S=2))


@pytest.mark.parametrize("kv", KINDS)
def test_attention_any_masks(dev, kv):
    """Masks of no tree: later tokens, not itself, nothing (zeros where there is no prefix either); fewer cached
    positions than tokens; bits of tokens that are not there."""
    r = np.random.RandomState(8)
    c = Case(dev, kv, [20, 9, 6, 4], [20, 5, 140, 0], 2, 64, seed=8)
    c.masks[:, 0] = r.randint(0, 1 << 62, c.N).astype(np.uint64)
    c.masks[3] = c.masks[21] = c.masks[30] = 0
    got = c.run()
    c.check(got)
    assert (got[3] == 0).all() and (got[c.start[3]:] == 0).all()


@pytest.mark.parametrize("kv", KINDS)
def test_attention_missing_pages(dev, kv):
    c = Case(dev, kv, [6, 18, 3], [400, 256, 64], 2, 64, seed=9, missing=[(0, 0), (0, 3), (1, 3), (2, 0)])
    got = c.run()
    c.check(got)
    assert (got[c.start[2]:c.start[3]] == 0).all()


@pytest.mark.parametrize("kv", KINDS)
def test_attention_large_scores(dev, kv):
    """The largest score keeps its weight at any magnitude."""
    c = Case(dev, kv, [18], [300], 2, 64, seed=10, sharp=200.0)
    c.check(c.run())


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("what", ["nan", "inf"])
def test_attention_bad_rows_of_others(dev, kv, what):
    """K, V and scales of tokens that a token does not attend never reach it; what attends them is not finite."""
    import torch
    c = Case(dev, kv, [40, 20], [200, 20], 2, 64, seed=11)
    bad = {0: 3, 1: 6}                                   # sequence: the token whose rows are bad
    value = float("nan") if what == "nan" else float("inf")
    for b, i in bad.items():
        pos = c.lens[b] - c.sizes[b] + i
        page, row = c.table[b][pos // c.R], pos % c.R
        if c.scale is not None:
            c.scale[page, :, :, row] = value
            if kv == "fp8":
                c.stored[page, :, :, row, 5] = 0x7F      # E4M3's NaN
        else:
            c.stored[page, 0, :, row, 2] = value
            c.stored[page, 1, :, row, 60] = -value
    got = c.run()
    clean = Case(dev, kv, c.sizes, c.lens, 2, 64, seed=11)
    for b, i in bad.items():
        for t in range(c.sizes[b]):
            at = c.start[b] + t
            if (int(c.masks[at, 0]) >> i) & 1:
                assert not np.isfinite(got[at]).all()
                got[at] = 0.0
                clean.q[at] = 0.0                        # (not compared)
            for h in range(2):
                k, v, ks, vs, ok = clean.rows(b, h)
                if (int(c.masks[at, 0]) >> i) & 1:
                    continue
                ref, bound = treeref.attend(c.q[at, 0, h].astype(np.float64), k, v, c.seen(b, t), ks, vs, kv)
                assert (np.abs(got[at, h] - ref) <= bound).all(), (b, t, h)
    # What lies past the last position is not read, whatever it is.
    c = Case(dev, kv, [5], [70], 1, 64, seed=12)
    page = c.table[0][1]
    if c.scale is not None:
        c.scale[page, :, :, 6:] = value
    else:
        c.stored[page, :, :, 6:] = value
    c.check(c.run())
    assert torch.cuda.is_available()


def test_attention_of_a_chain_is_that_of_tokens(dev):
    """paged_decode_tokens' drafts are the tree whose parents are the tokens before."""
    import torch
    kvattn = _kv()
    c = Case(dev, "int4", [8, 3], [333, 90], 2, 64, seed=13)
    c.parents = np.concatenate([np.arange(-1, 7), np.arange(-1, 2)]).astype(np.int32)
    c.masks, _ = treeref.masks(c.start, c.parents, 1)
    got = c.run(spare=0)
    c.check(got)
    qkv = torch.from_numpy(c.q).to(torch.bfloat16).to(dev)
    out = torch.zeros((c.N, 2, HS), dtype=torch.bfloat16, device=dev)
    cache = kvattn.PagedCache(c.stored.to(dev), _dev(c.table, dev), c.max_pages, 64, c.P, c.scale.to(dev))
    ws = kvattn.Workspace(c.N, 2, c.max_pages * 64)
    kvattn.paged_decode_tokens(out, qkv, cache, _dev(c.start, dev), _dev(np.array(c.lens, dtype=np.int32), dev), 2, c.N, 2, HS,
                               kv_dtype="int4", max_new=8, **ws.kwargs())
    c.check(out.double().cpu().numpy())


@pytest.mark.parametrize("kv", ["bf16", "fp4"])
def test_attention_more_tokens_than_max_new(dev, kv):
    """A sequence with more tokens than max_new has the first max_new computed."""
    c = Case(dev, kv, [50, 4], [300, 90], 1, 64, seed=14)
    c.check(c.run(max_new=10), tokens=10)


def test_attention_long_and_many(dev):
    """A long sequence whose segments join, and more sequences than CUs."""
    c = Case(dev, "bf16", [30], [6000], 1, 256, seed=15)
    c.check(c.run())
    c = Case(dev, "int8", [2] * 300, [70 + i % 50 for i in range(300)], 1, 64, seed=16)
    c.check(c.run())


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("NH", [1, 3])
def test_keep(dev, kv, NH):
    import torch
    kvattn = _kv()
    r = np.random.RandomState(20)
    sizes = [12, 0, 1, 30, 9, 5]
    paths = [[0, 2, 3, 7, 11], [], [0], [0, 1] + list(range(3, 25)), [0, 4, 8], [0, 3, 2, 4]]    # (the last: up to 2)
    start = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    N, R, P = int(start[-1]), 64, 4
    path = np.full(N, -1, dtype=np.int32)
    for t0, p in zip(start, paths):
        path[t0:t0 + len(p)] = p
    slots = r.permutation(P * R)[:N].astype(np.int64)
    slots[start[4] + 8] = -1                             # a step without a place
    stored, scale = treeref.encode(r.standard_normal((P, 2, NH, R, HS)).astype(np.float32), kv)
    want, want_s = stored.clone(), None if scale is None else scale.clone()
    for b, p in enumerate(paths):
        last = -1
        for d, v in enumerate(p):
            if not (v > last and v >= d and v < sizes[b]):
                break
            last = v
            src, dst = slots[start[b] + v], slots[start[b] + d]
            if src >= 0 and dst >= 0:
                want[dst // R, :, :, dst % R] = stored[src // R, :, :, src % R]
                if scale is not None:
                    want_s[dst // R, :, :, dst % R] = scale[src // R, :, :, src % R]
    pages, scales = stored.to(dev), None if scale is None else scale.to(dev)
    cache = kvattn.PagedCache(pages, None, 1, R, P, scales)
    kvattn.paged_keep(cache, _dev(slots, dev), _dev(path, dev), _dev(start, dev), len(sizes), N, NH, HS, kv_dtype=kv)
    assert torch.equal(pages.cpu().view(torch.uint8), want.view(torch.uint8))
    if scale is not None:
        assert torch.equal(scales.cpu(), want_s)


@pytest.mark.parametrize("kv", ["f32", "int4"])
def test_pools_beyond_32_bits(dev, kv):
    """Pages whose bytes lie past 2^32: the same rows as in a small pool, read and moved."""
    import torch
    kvattn = _kv()
    NH, R, n = 12, 256, 5
    c = Case(dev, kv, [n], [700], NH, R, seed=60)
    near = c.stored.to(dev)
    page_bytes = near[0].numel() * near.element_size()
    extra = (1 << 32) // page_bytes + 1
    far = torch.zeros((extra + c.P,) + tuple(near.shape[1:]), dtype=near.dtype, device=dev)
    far[extra:] = near
    scales = far_scales = None
    if c.scale is not None:
        scales = c.scale.to(dev)
        far_scales = torch.zeros((extra + c.P,) + tuple(scales.shape[1:]), device=dev)
        far_scales[extra:] = scales
    start, lens, masks = _dev(c.start, dev), _dev(np.array([700], dtype=np.int32), dev), _dev(c.masks, dev)
    qkv = torch.from_numpy(c.q).to(c.act).to(dev)
    ws = kvattn.Workspace(c.N, NH, c.max_pages * R)
    path = torch.tensor([0, 2, 4, -1, -1], dtype=torch.int32, device=dev)
    outs = []
    for pages, sc, first in ((near, scales, 0), (far, far_scales, extra)):
        cache = kvattn.PagedCache(pages, _dev(c.table + first, dev).int(), c.max_pages, R, first + c.P, sc)
        out = torch.zeros((c.N, NH, HS), dtype=c.act, device=dev)
        kvattn.paged_decode_tree(out, qkv, cache, start, lens, masks, 1, c.N, NH, HS, kv_dtype=kv, max_new=n, **ws.kwargs())
        outs.append(out)
        slots = torch.tensor([(int(c.table[0, t // R]) + first) * R + t % R for t in range(695, 700)], device=dev)
        kvattn.paged_keep(cache, slots, path, start, 1, c.N, NH, HS, kv_dtype=kv)
    assert torch.equal(outs[0], outs[1])
    assert torch.equal(far[extra:].view(torch.uint8), near.view(torch.uint8)) and not far[:extra].any()
    assert not torch.equal(near.cpu().view(torch.uint8), c.stored.view(torch.uint8))


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_captured_calls_and_other_streams(dev, kv):
    """Two graphs and eager calls on one workspace, ordered, with lengths that change between replays."""
    import torch
    kvattn = _kv()
    NH, R = 5, 64
    c = Case(dev, kv, [20, 3, 33], [1500, 40, 900], NH, R, seed=61)
    cache = kvattn.PagedCache(c.stored.to(dev), _dev(c.table, dev), c.max_pages, R, c.P, None if c.scale is None else c.scale.to(dev))
    start, masks = _dev(c.start, dev), _dev(c.masks, dev)
    lens = _dev(np.array(c.lens, dtype=np.int32), dev)
    qkv = torch.from_numpy(c.q).to(c.act).to(dev)
    ws = kvattn.Workspace(c.N, NH, c.max_pages * R, S=6)
    outs = [torch.zeros((c.N, NH, HS), dtype=c.act, device=dev) for _ in range(3)]

    def call(out):
        kvattn.paged_decode_tree(out, qkv, cache, start, lens, masks, 3, c.N, NH, HS, kv_dtype=kv, max_new=33, S=6, **ws.kwargs())

    call(outs[0])
    torch.cuda.synchronize()
    graphs = []
    for out in outs[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(out)
    side = torch.cuda.Stream()
    for step in range(4):
        lens.copy_(_dev(np.array(c.lens, dtype=np.int32) - 7 * step, dev))
        for out in outs:
            out.fill_(9.0)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(outs[2])
        torch.cuda.current_stream().wait_stream(side)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[2]) and not (outs[2] == 9.0).any()
