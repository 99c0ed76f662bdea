"""Verification of trees of drafted tokens against a walk in 64 bits (treeref.walk)."""
import numpy as np
import pytest

import treeref

pytestmark = pytest.mark.gpu


def _kv():
    from cuda_gpt2_inference_amd import kvattn
    return kvattn


def _i32(x, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(dev)


def _f32(x, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(dev)


def _workspace(dev, B, V):
    import torch
    kvattn = _kv()
    ws = torch.empty(kvattn.verify_workspace_bytes(B, V), dtype=torch.uint8, device=dev)
    kvattn.workspace_init(ws, ws.numel())
    return ws


def _case(r, sizes, V, stride, dtype, wild=False):
    start, parents = treeref.forest(r, sizes, wild)
    N = len(parents)
    z = 2.5 * r.standard_normal((N, V))
    p = np.full((N, stride), np.nan, dtype=np.float32)          # what lies behind the vocabulary is not read
    e = np.exp(z - z.max(-1, keepdims=True))
    p[:, :V] = e / e.sum(-1, keepdims=True)
    if dtype == "bf16":
        p = treeref.bf16(p)
    tokens = np.zeros(N, dtype=np.int32)
    for t0, n in zip(start, sizes):
        tokens[t0:t0 + n] = r.randint(0, V, n)
        for i in range(1, n):
            if 0 <= parents[t0 + i] < i:
                row = np.float64(p[t0 + parents[t0 + i], :V]) ** 1.5
                tokens[t0 + i] = r.choice(V, p=row / row.sum())
    return start, parents, p, tokens, r.rand(N).astype(np.float32), r.rand(len(sizes)).astype(np.float32)


def _check(dev, start, parents, p, tokens, u, draw, V, dtype="f32", offset=0, ws=None, in_place=False):
    import torch
    kvattn = _kv()
    N, stride = p.shape
    B = len(start) - 1
    td = torch.float32 if dtype == "f32" else torch.bfloat16
    flat = torch.empty(p.size + offset, dtype=td, device=dev)
    flat[offset:] = torch.from_numpy(p).view(-1).to(td)
    lens = np.arange(B) * 7 + 300
    out = torch.full((N + 4,), -2, dtype=torch.int32, device=dev)
    tree = _i32(np.concatenate([tokens, [0] * 4]), dev)
    if in_place:
        out = tree
        out[N:] = -2
    path, counts, kept = (torch.full((k,), -2, dtype=torch.int32, device=dev) for k in (N + 4, B + 2, B + 2))
    ws = _workspace(dev, B, V) if ws is None else ws
    kvattn.verify_tree(out, path, counts, flat[offset:], tree, _i32(parents, dev), _f32(u, dev), _f32(draw, dev), _i32(start, dev),
                       B, N, V, lens=_i32(lens, dev), kept=kept, row_stride=stride, dtype=dtype, workspace=ws,
                       workspace_nbytes=ws.numel())
    out, path, counts, kept = (x.cpu().numpy() for x in (out, path, counts, kept))
    assert (out[N:] == -2).all() and (path[N:] == -2).all() and (counts[B:] == -2).all() and (kept[B:] == -2).all()
    assert not ws.any()                                          # left as it was found
    deepest = 0
    for b in range(B):
        t0, n = int(start[b]), int(start[b + 1] - start[b])
        if n == 0:
            assert counts[b] == 0 and kept[b] == lens[b]
            continue
        want, way = treeref.walk(p[:, :V], tokens, parents, u, draw[b], t0, n)
        assert out[t0:t0 + n].tolist() == want + [-1] * (n - len(want)), b
        assert path[t0:t0 + n].tolist() == way + [-1] * (n - len(way)), b
        assert counts[b] == len(want) and kept[b] == lens[b] - n + len(way)
        deepest = max(deepest, len(way))
    return deepest


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sizes,V,stride", [
    ([1], 1, 1), ([2, 1, 0, 5], 7, 8), ([26], 50257, 50304), ([64, 3, 65, 0, 1, 17], 300, 301), ([256, 300, 129], 1025, 1028),
    ([16] * 40, 2000, 2000), ([4] * 700, 50, 52)])
def test_walk(dev, dtype, sizes, V, stride):
    r = np.random.RandomState(sum(sizes) + V)
    for wild in (False, True):
        _check(dev, *_case(r, sizes, V, stride, dtype, wild), V, dtype)


def test_walks_go_deep(dev):
    """Numbers that accept the first child wherever there is one (how deep that goes is the tree's affair), and numbers
    that accept less; a chain to its end."""
    r = np.random.RandomState(3)
    start, parents, p, tokens, u, draw = _case(r, [200, 40], 20, 20, "f32")
    deep = _check(dev, start, parents, p, tokens, np.zeros_like(u), draw, 20)
    assert _check(dev, start, parents, p, tokens, np.full_like(u, 0.9999999), draw, 20) < deep
    parents = np.concatenate([np.arange(-1, 199), np.arange(-1, 39)]).astype(np.int32)
    assert _check(dev, start, parents, p, tokens, np.zeros_like(u), draw, 20) == 200


@pytest.mark.parametrize("offset", [0, 1, 2])
def test_unaligned_rows(dev, offset):
    r = np.random.RandomState(4)
    _check(dev, *_case(r, [9, 20], 3000, 3001 + offset, "bf16"), 3000, "bf16", offset=offset)
    _check(dev, *_case(r, [9, 20], 3000, 3001 + offset, "f32"), 3000, "f32", offset=offset)


def test_strange_rows(dev):
    """Children that are one token, of ids that are none, that take the whole mass; rows without mass or with NaN,
    infinities, negative numbers."""
    r = np.random.RandomState(5)
    V = 40
    start, parents, p, tokens, u, draw = _case(r, [12] * 30, V, V, "f32")
    for b in range(30):
        t0 = start[b]
        kind = b % 6
        if kind == 0:
            parents[t0 + 1:t0 + 12] = 0
            tokens[t0 + 1:t0 + 12] = r.randint(0, 3, 11)         # the same few tokens again
        elif kind == 1:
            tokens[t0 + 1:t0 + 12] = r.choice([-1, V, V + 5, 1 << 30, -(1 << 31), 3], 11)
        elif kind == 2:
            p[t0:t0 + 12] = 0.0
            p[t0:t0 + 12, 5] = 0.75                              # a sum below one, all of it the children's
            tokens[t0 + 1:t0 + 12] = 5
            u[t0:t0 + 12] = r.choice([0.7, 0.8], 12)
        elif kind == 3:
            p[t0:t0 + 12] = 0.0
        elif kind == 4:
            p[t0:t0 + 12, ::3] = r.choice([np.nan, np.inf, -np.inf, -2.0], (12, len(range(0, V, 3))))
        else:
            draw[b] = 0.0
            u[t0:t0 + 12] = 0.0
    _check(dev, start, parents, p, tokens, u, draw, V)


def test_workspace_serves_both_verifications(dev):
    """One workspace of the largest size, other B and V, trees and chains in turn; tokens in the tree's place."""
    import torch
    kvattn = _kv()
    r = np.random.RandomState(6)
    ws = _workspace(dev, 64, 50257)
    for sizes, V in (([30], 50257), ([3] * 64, 900), ([8, 8], 20000)):
        _check(dev, *_case(r, sizes, V, V, "f32"), V, ws=ws, in_place=True)
        p = torch.softmax(torch.randn(4, V, device=dev), -1)
        tokens, counts = torch.zeros(4, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
        kvattn.verify_drafts(tokens, counts, p, _i32([1, 2, 3, 0], dev), _f32([0.5] * 4, dev), _i32([0, 4], dev), 1, 4, V,
                             workspace=ws, workspace_nbytes=ws.numel())
        assert not ws.any() and int(counts[0]) >= 1


def test_no_tokens(dev):
    import torch
    kvattn = _kv()
    ws = _workspace(dev, 3, 100)
    counts, kept = (torch.full((3,), 9, dtype=torch.int32, device=dev) for _ in range(2))
    kvattn.verify_tree(None, None, counts, None, None, None, None, None, _i32([0, 0, 0, 0], dev), 3, 0, 100, lens=_i32([4, 5, 6], dev),
                       kept=kept, workspace=ws, workspace_nbytes=ws.numel())
    assert counts.tolist() == [0, 0, 0] and kept.tolist() == [4, 5, 6]
