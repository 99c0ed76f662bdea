"""Steps of a server that verifies trees of drafted tokens: projections on 4-bit weights, pages from lengths, K and V by
slot, attention of the trees, logits with penalties and grammar masks, the walk, and the accepted rows next to the
prefix.  Eager and from one captured graph, every replay against the eager step and the walk against a restatement."""
import numpy as np
import pytest

import treeref

pytestmark = pytest.mark.gpu

NH, C, V = 2, 128, 20          # few tokens, so that a tree of any holds some that are accepted
B, R, MAX_PAGES, NUM_PAGES = 4, 64, 4, 16
MAX_NEW, MAX_TOKENS = 12, 40
HISTORY = 64


class Server:
    def __init__(self, dev, kv, seed):
        import torch
        from cuda_gpt2_inference_amd import kvattn
        self.k, self.kv = kvattn, kv
        z = lambda *s, d=torch.int32: torch.zeros(s, dtype=d, device=dev)       # noqa: E731
        f, h = torch.float32, torch.bfloat16
        self.act = f if kv == "f32" else h
        store = {"f32": f, "bf16": h}.get(kv, torch.uint8)
        width = 32 if kv in ("int4", "fp4") else 64
        self.cache = kvattn.PagedCache(z(NUM_PAGES, 2, NH, R, width, d=store), z(B, MAX_PAGES), MAX_PAGES, R, NUM_PAGES,
                                       None if kv in ("f32", "bf16") else z(NUM_PAGES, 2, NH, R, d=f))
        self.pool = kvattn.paged_pool(NUM_PAGES, device=dev)
        self.held, self.kept, self.fresh, self.lens, self.start = z(B), z(B), z(B), z(B), z(B + 1)
        self.slots = z(MAX_TOKENS, d=torch.int64)
        self.masks, self.positions = z(MAX_TOKENS, 1, d=torch.int64), z(MAX_TOKENS)
        self.parents, self.tree = z(MAX_TOKENS), z(MAX_TOKENS)
        self.x = z(MAX_TOKENS, C, d=h)
        self.qkv = z(MAX_TOKENS, 3, NH, 64, d=self.act)
        self.att, self.att16 = z(MAX_TOKENS, NH, 64, d=self.act), z(MAX_TOKENS, NH * 64, d=h)
        self.logits, self.probs = z(MAX_TOKENS, V, d=f), z(MAX_TOKENS, V, d=f)
        g = torch.Generator().manual_seed(seed)
        w = lambda m, c: (0.3 * torch.randn(m, c, generator=g)).to(h).to(dev)    # noqa: E731
        self.wqkv = kvattn.w4_quantize(w(3 * NH * 64, C), 3 * NH * 64, C, 32, w_dtype="int4")
        self.wte = kvattn.w4_quantize(w(V, NH * 64), V, NH * 64, 64, w_dtype="fp4")
        self.history, self.history_len = z(B, HISTORY), z(B)
        self.allowed, self.allowed_of = z(2, (V + 31) // 32), z(MAX_TOKENS)
        self.allowed[0] = -1
        self.allowed[1, ::2] = -1
        self.u, self.draw = z(MAX_TOKENS, d=f), z(B, d=f)
        self.tokens, self.path, self.counts = z(MAX_TOKENS), z(MAX_TOKENS), z(B)
        t = lambda *x: torch.tensor(x, device=dev, dtype=f)                       # noqa: E731
        self.rules = kvattn.LogitRules(
            history=self.history, history_len=self.history_len, max_history=HISTORY, tokens=self.tree, masks=self.masks, mask_words=1,
            repetition=t(1.0, 1.2, 1.5, 1.1), frequency=t(0.1, 0.0, 0.3, 0.2), presence=t(0.0, 0.2, 0.1, 0.0),
            temperature=t(1.0, 0.7, 0.0, 1.3), allowed=self.allowed, allowed_of=self.allowed_of, num_allowed=2,
            allowed_stride=self.allowed.shape[1])
        self.ws = kvattn.Workspace(MAX_TOKENS, NH, MAX_PAGES * R)
        self.vws = torch.empty(kvattn.verify_workspace_bytes(B, V), dtype=torch.uint8, device=dev)
        kvattn.workspace_init(self.vws, self.vws.numel())

    def issue(self):
        k, N = self.k, MAX_TOKENS
        k.gemv_w4(self.qkv, self.wqkv, self.x, N, 3 * NH * 64, C, group=32, w_dtype="int4", out_dtype="f32" if self.kv == "f32" else "bf16")
        k.paged_reserve(self.cache, self.pool, self.held, self.kept, self.fresh, B, lens=self.lens, token_start=self.start,
                        slot_map=self.slots, max_tokens=N)
        k.paged_store(self.cache, self.qkv, self.slots, N, NH, 64, kv_dtype=self.kv)
        k.tree_masks(self.masks, self.parents, self.start, B, N, positions=self.positions, lens=self.lens)
        k.paged_decode_tree(self.att, self.qkv, self.cache, self.start, self.lens, self.masks, B, N, NH, 64, kv_dtype=self.kv,
                            max_new=MAX_NEW, **self.ws.kwargs())
        self.att16.copy_(self.att.view(N, NH * 64))
        k.gemv_w4(self.logits, self.wte, self.att16, N, V, NH * 64, group=64, w_dtype="fp4", out_dtype="f32")
        k.process_logits(self.probs, self.logits, self.rules, self.start, B, N, V)
        k.verify_tree(self.tokens, self.path, self.counts, self.probs, self.tree, self.parents, self.u, self.draw, self.start, B, N,
                      V, lens=self.lens, kept=self.kept, workspace=self.vws, workspace_nbytes=self.vws.numel())
        k.paged_keep(self.cache, self.slots, self.path, self.start, B, N, NH, 64, kv_dtype=self.kv)

    def load(self, fresh, start, parents, tree, x, u, draw, lines):
        import torch
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a))                   # noqa: E731
        self.fresh.copy_(t(fresh))
        n = len(parents)
        self.parents[:n] = t(parents).to(self.parents.device)
        self.tree[:n] = t(tree).to(self.tree.device)
        self.x.copy_(t(x))
        self.u.copy_(t(u))
        self.draw.copy_(t(draw))
        self.allowed_of.copy_(t(lines))

    def rows(self, b, positions):
        """Stored rows of a sequence's positions, scales behind them."""
        import torch
        page = self.cache.block_table[b][positions // R].long()
        row = (positions % R).long()
        out = self.cache.pages[page, :, :, row].contiguous().view(torch.uint8).flatten(1)
        if self.cache.page_scales is not None:
            out = torch.cat([out, self.cache.page_scales[page, :, :, row].contiguous().view(torch.uint8).flatten(1)], dim=1)
        return out.cpu()


@pytest.mark.parametrize("kv", ["f32", "bf16", "int8", "fp8", "int4", "fp4"])
def test_steps(dev, kv):
    import torch
    r = np.random.RandomState(50)
    s, twin = Server(dev, kv, 1), Server(dev, kv, 1)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        twin.issue()
    text = [[int(r.randint(V))] for _ in range(B)]                               # accepted tokens; the last has no row yet
    cached = [None] * B                                                           # rows of the kept positions
    moved = 0
    for step in range(14):
        fresh = r.randint(0 if step else 1, MAX_NEW + 1, B).astype(np.int32)
        while fresh.sum() > MAX_TOKENS:
            fresh[fresh.argmax()] -= 1
        start, parents = treeref.forest(r, fresh.tolist())
        tree = r.randint(0, V, len(parents)).astype(np.int32)
        # The root is the token that the last step drew.
        for b in range(B):
            if fresh[b]:
                tree[start[b]] = text[b][-1]
        x = treeref.bf16(r.standard_normal((MAX_TOKENS, C)))
        u, draw = (r.rand(MAX_TOKENS) ** 3).astype(np.float32), r.rand(B).astype(np.float32)
        lines = r.randint(-1, 2, MAX_TOKENS).astype(np.int32)
        kept_before = s.kept.cpu().numpy().copy()
        for z in (s, twin):
            z.load(fresh, start, parents, tree, x, u, draw, lines)
            z.history.zero_()
            for b in range(B):
                h = torch.tensor(text[b][:-1][-HISTORY:], dtype=torch.int32)
                z.history[b, :len(h)] = h.to(dev)
                z.history_len[b] = len(h)
        s.issue()
        graph.replay()
        torch.cuda.synchronize()
        for name in ("tokens", "path", "counts", "kept", "lens", "start", "held", "slots"):
            assert torch.equal(getattr(s, name), getattr(twin, name)), (step, name)
        N = len(parents)
        assert torch.equal(s.probs[:N], twin.probs[:N]) and torch.equal(s.att[:N], twin.att[:N])
        assert torch.equal(s.cache.pages.view(torch.uint8), twin.cache.pages.view(torch.uint8))
        assert s.start.tolist() == start.tolist()
        p, got, path, kept, lens = (t.cpu().numpy() for t in (s.probs, s.tokens, s.path, s.kept, s.lens))
        for b in range(B):
            t0, n = int(start[b]), int(fresh[b])
            assert lens[b] == kept_before[b] + n
            if n == 0:
                assert kept[b] == lens[b]
                continue
            want, way = treeref.walk(p, tree, parents, u, draw[b], t0, n)
            assert got[t0:t0 + len(want)].tolist() == want and path[t0:t0 + len(way)].tolist() == way
            assert kept[b] == kept_before[b] + len(way)
            text[b] += want
            moved += way != list(range(len(way)))
            # The cache: what was kept stays, then the path's rows as they were stored.
            codes, scale = treeref.encode(s.qkv[t0:t0 + n, 1:].float().cpu().numpy(), kv)
            new = codes[way].contiguous().view(torch.uint8).flatten(1)
            if scale is not None:
                new = torch.cat([new, scale[way].contiguous().view(torch.uint8).flatten(1)], dim=1)
            cached[b] = new if cached[b] is None else torch.cat([cached[b], new])
            assert torch.equal(s.rows(b, torch.arange(int(kept[b]), device=dev)), cached[b]), (step, b)
        if max(len(t) for t in text) > 180:
            break
    assert moved > 0
