"""Steps of speculative decoding as a server makes them: pages from lengths, K and V by slot, attention of
the drafted tokens over the 4-bit pages, logits, verification, and the next step from what was kept.
Every step against restatements that never see the pages (kv4ref); then the same steps from one
captured graph."""
import numpy as np
import pytest

import kv4ref
from kv4ref import HS

pytestmark = pytest.mark.gpu

NH, V = 2, 300
B, R, MAX_PAGES, NUM_PAGES = 5, 64, 4, 6
MAX_NEW, MAX_TOKENS = 6, 24


class Server:
    """The device side of a step; `issue` is what a graph may hold."""

    def __init__(self, dev, kv, seed):
        import torch
        from cuda_gpt2_inference_amd import kvattn
        self.kvattn, self.kv = kvattn, kv
        z = lambda *s, d=torch.int32: torch.zeros(s, dtype=d, device=dev)       # noqa: E731
        self.cache = kvattn.PagedCache(z(NUM_PAGES, 2, NH, R, HS // 2, d=torch.uint8), z(B, MAX_PAGES), MAX_PAGES, R,
                                       NUM_PAGES, torch.full((NUM_PAGES, 2, NH, R), float("nan"), device=dev))
        self.pool = kvattn.paged_pool(NUM_PAGES, device=dev)
        self.held, self.kept, self.fresh = z(B), z(B), z(B)
        self.lens, self.start = z(B), z(B + 1)
        self.slots, self.positions = z(MAX_TOKENS, d=torch.int64), z(MAX_TOKENS)
        self.qkv = z(MAX_TOKENS, 3, NH, HS, d=torch.bfloat16)
        self.att = z(MAX_TOKENS, NH, HS, d=torch.bfloat16)
        g = torch.Generator().manual_seed(seed)
        self.W = (torch.randn(V, NH * HS, generator=g) * 0.5).to(torch.bfloat16).to(dev)
        self.logits = z(MAX_TOKENS, V, d=torch.float32)
        self.probs = z(MAX_TOKENS, V, d=torch.float32)
        self.q = z(MAX_TOKENS, V, d=torch.float32)
        self.drafts, self.u = z(MAX_TOKENS), z(MAX_TOKENS, d=torch.float32)
        self.tokens, self.counts = z(MAX_TOKENS), z(B)
        self.ws = kvattn.Workspace(MAX_TOKENS, NH, MAX_PAGES * R)
        n = kvattn.verify_workspace_bytes(B, V)
        self.vws = torch.empty(n, dtype=torch.uint8, device=dev)
        kvattn.workspace_init(self.vws, n)

    def issue(self):
        import torch
        k = self.kvattn
        k.paged_reserve(self.cache, self.pool, self.held, self.kept, self.fresh, B, lens=self.lens, token_start=self.start,
                        slot_map=self.slots, positions=self.positions, max_tokens=MAX_TOKENS)
        k.paged_store(self.cache, self.qkv, self.slots, MAX_TOKENS, NH, HS, kv_dtype=self.kv)
        k.paged_decode_tokens(self.att, self.qkv, self.cache, self.start, self.lens, B, MAX_TOKENS, NH, HS,
                              kv_dtype=self.kv, max_new=MAX_NEW, **self.ws.kwargs())
        k.gemv(self.logits, self.W, self.att, MAX_TOKENS, V, NH * HS, w_dtype="bf16", out_dtype="f32")
        self.probs.copy_(torch.softmax(self.logits, dim=-1))
        k.verify_drafts(self.tokens, self.counts, self.probs, self.drafts, self.u, self.start, B, MAX_TOKENS, V,
                        draft_probs=self.q, workspace=self.vws, workspace_nbytes=self.vws.numel())


def _inputs(r, kept):
    """A step's fresh counts, and rows of q, k, v, drafts and random numbers (host)."""
    ended = r.rand(B) < 0.01
    kept = np.where(ended, 0, kept)
    fresh = np.where(r.rand(B) < 0.15, 0, r.randint(1, MAX_NEW + 1, B))
    fresh = np.where(kept == 0, MAX_NEW, fresh)                              # a new request's prompt comes in chunks
    fresh = np.minimum(fresh, MAX_PAGES * R - kept)
    while fresh.sum() > MAX_TOKENS:
        fresh[fresh.argmax()] -= 1
    qkv = r.standard_normal((MAX_TOKENS, 3, NH, HS)).astype(np.float32)
    z = r.standard_normal((MAX_TOKENS, V))
    q = np.exp(z) / np.exp(z).sum(-1, keepdims=True)
    drafts = np.array([r.choice(V, p=row) for row in q])
    return kept, fresh, qkv, q.astype(np.float32), drafts, r.rand(MAX_TOKENS).astype(np.float32)


def _load(s, kept, fresh, qkv, q, drafts, u):
    import torch
    t = lambda x, d: torch.from_numpy(np.ascontiguousarray(x)).to(d)      # noqa: E731
    s.kept.copy_(t(kept, torch.int32))
    s.fresh.copy_(t(fresh, torch.int32))
    s.qkv.copy_(t(qkv, torch.bfloat16))
    s.q.copy_(t(q, torch.float32))
    s.drafts.copy_(t(drafts, torch.int32))
    s.u.copy_(t(u, torch.float32))


@pytest.mark.parametrize("kv", ["int4", "fp4"])
def test_steps(dev, kv):
    import torch
    r = np.random.RandomState(40)
    s = Server(dev, kv, 1)
    twin = Server(dev, kv, 1)                       # the same steps from one captured graph
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        twin.issue()
    model = kv4ref.Pool(NUM_PAGES)
    table, held = np.zeros((B, MAX_PAGES), np.int32), np.zeros(B, np.int64)
    rows = [[] for _ in range(B)]                   # [K codes, K scales, V codes, V scales] of every kept position
    kept = np.zeros(B, np.int64)
    refused = 0
    for step in range(80):
        inp = _inputs(r, kept)
        kept, fresh, qkv = inp[0], inp[1], inp[2]
        for x in (s, twin):
            _load(x, *inp)
        s.issue()
        graph.replay()
        torch.cuda.synchronize()
        start = np.concatenate([[0], np.cumsum(fresh)])
        held, lens, want_start, slots, pos = model.reserve(table, R, held, kept, fresh, MAX_TOKENS)
        assert np.array_equal(want_start, start)
        assert np.array_equal(s.cache.block_table.cpu().numpy(), table) and s.pool[:2].tolist() == [model.head, model.count]
        assert np.array_equal(s.held.cpu().numpy(), held) and np.array_equal(s.lens.cpu().numpy(), lens)
        codes, scale = kv4ref.encode(torch.from_numpy(qkv[:, 1:]).to(torch.bfloat16).float().numpy(), kv)
        att = s.att.float().cpu().numpy()
        qbf = torch.from_numpy(qkv[:, 0]).to(torch.bfloat16).float().numpy()
        for b in range(B):
            del rows[b][kept[b]:]
            granted = lens[b] == kept[b] + fresh[b]
            refused += not granted
            for i in range(fresh[b] if granted else 0):
                t = start[b] + i
                rows[b].append((codes[t], scale[t]))
                for h in range(NH):
                    c = np.stack([x[0][:, h] for x in rows[b]], 1)
                    sc = np.stack([x[1][:, h] for x in rows[b]], 1)
                    n = len(rows[b])
                    k, v = (kv4ref.decode(c[p], sc[p], kv) for p in (0, 1))
                    ref, wv = kv4ref.attend(qbf[t, h].astype(np.float64), k, v, n)
                    lim = kv4ref.bound(ref, wv, qbf[t, h], sc[0], sc[1], kv, n)
                    assert (np.abs(att[t, h] - ref) <= lim).all(), (step, b, i, h)
        tokens, counts = kv4ref.verify(s.probs.double().cpu().numpy(), inp[3].astype(np.float64), inp[4], inp[5], start, V)
        n = start[-1]
        assert np.array_equal(s.tokens.cpu().numpy()[:n], tokens[:n]) and np.array_equal(s.counts.cpu().numpy(), counts)
        for name in ("att", "tokens", "counts", "held", "lens", "start", "slots", "pool"):
            a, b2 = getattr(s, name), getattr(twin, name)
            assert torch.equal(a[:n] if name in ("att", "tokens") else a, b2[:n] if name in ("att", "tokens") else b2), name
        assert torch.equal(s.cache.pages, twin.cache.pages)
        kept = np.where(lens == kept + fresh, kept + counts, kept)
        kept = np.minimum(kept, held)
    assert refused > 0, "the pool is small enough that some step was refused"


def _next_kept(lens, kept, fresh, counts):
    """What a request keeps after a step: a granted one its tokens up to the last emitted one's place, a refused one,
    for whose rows the step's other calls computed nothing that counts, what it had."""
    import torch
    return torch.where(lens == kept + fresh, kept + counts, kept)


def _last(lens, kept, fresh, counts):
    return lens - fresh + counts                    # right for the granted ones alone


@pytest.mark.parametrize("rule", [_next_kept, _last])
@pytest.mark.parametrize("kv", ["int4", "fp4"])
def test_refused_requests_lose_nothing(dev, kv, rule):
    """Steps whose next kept positions are computed on the device, over a pool that is too small: every position that
    was kept holds the row that was accepted for it, however often its request was refused since.  (A rule that
    takes the rows of refused requests for accepted ones is caught.)"""
    import torch
    r = np.random.RandomState(41)
    s = Server(dev, kv, 2)
    rows = [[] for _ in range(B)]                   # (step, token row) of every kept position
    log, refused, wrong = [], 0, False
    kept = torch.zeros(B, dtype=torch.int32, device=dev)
    for step in range(100):
        wrong = kept.tolist() != [len(x) for x in rows]
        if wrong:
            break
        if step in (60, 80):
            kept[step // 20], rows[step // 20] = 0, []          # one ends, and its pages go to others
        k = kept.cpu().numpy()
        fresh = np.minimum(r.randint(1, 5, B), MAX_PAGES * R - k)
        qkv = r.standard_normal((MAX_TOKENS, 3, NH, HS)).astype(np.float32)
        q = np.full((MAX_TOKENS, V), 1 / V, np.float32)
        _load(s, k, fresh, qkv, q, r.randint(0, V, MAX_TOKENS), 0.2 * r.rand(MAX_TOKENS).astype(np.float32))
        s.issue()
        start = np.concatenate([[0], np.cumsum(fresh)])
        granted, counts = (s.lens == kept + s.fresh).cpu().numpy(), s.counts.cpu().numpy()
        refused += int((~granted).sum())
        log.append(torch.from_numpy(qkv[:, 1:]).to(torch.bfloat16).float().numpy())
        for b in np.nonzero(granted)[0]:
            rows[b] += [(step, start[b] + i) for i in range(counts[b])]
        kept = rule(s.lens, kept, s.fresh, s.counts)
    if rule is _last:
        assert wrong
        return
    assert not wrong and refused > 5 and sum(map(len, rows)) > 100
    k = kept.cpu().numpy()
    table = s.cache.block_table.cpu().numpy()
    for b in range(B):
        assert len(rows[b]) == k[b] <= int(s.held[b])
        if not rows[b]:
            continue
        pos = np.arange(k[b])
        slots = torch.from_numpy(table[b, pos // R].astype(np.int64) * R + pos % R).to(dev)
        back = torch.zeros(k[b], 2, NH, HS, dtype=torch.bfloat16, device=dev)
        s.kvattn.paged_load(back, s.cache, slots, int(k[b]), NH, HS, kv_dtype=kv)
        codes, scale = kv4ref.encode(np.stack([log[t][row] for t, row in rows[b]]), kv)
        want = kv4ref.decode(codes, np.ones_like(scale), kv).astype(np.float32) * scale[..., None]
        assert torch.equal(back.cpu(), torch.from_numpy(want).to(torch.bfloat16)), b


def test_pages_and_rows_on_another_stream(dev):
    """Current stream not the default one: every call goes to it, in order."""
    import torch
    from cuda_gpt2_inference_amd import kvattn
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fresh = [70, 0, 3, 64, 65, 128]
        b, n, P, N = len(fresh), 4, 20, sum(fresh)
        z = lambda *s, d=torch.int32: torch.zeros(s, dtype=d, device=dev)       # noqa: E731
        cache = kvattn.PagedCache(z(P, 2, NH, R, HS, d=torch.bfloat16), z(b, n), n, R, P)
        pool, lens, start, slots = kvattn.paged_pool(P, device=dev), z(b), z(b + 1), z(N, d=torch.int64)
        kvattn.paged_reserve(cache, pool, z(b), z(b), torch.tensor(fresh, dtype=torch.int32, device=dev), b, lens=lens,
                             token_start=start, slot_map=slots, max_tokens=N)
        assert lens.tolist() == fresh and start[-1] == N and len(set(slots.tolist())) == N and slots.min() >= 0
        qkv = torch.randn(N, 3, NH, HS, device=dev).to(torch.bfloat16)
        kvattn.paged_store(cache, qkv, slots, N, NH, HS, kv_dtype="bf16")
        back = torch.zeros(N, 2, NH, HS, dtype=torch.bfloat16, device=dev)
        kvattn.paged_load(back, cache, slots, N, NH, HS, kv_dtype="bf16")
        assert torch.equal(back, qkv[:, 1:])
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("kv", ["int4", "fp4"])
def test_decode_on_another_stream(dev, kv):
    import torch
    from cuda_gpt2_inference_amd import kvattn
    from test_gpu_kv4 import Case, _dev, _qkv
    case = Case(kv, 1, 2, 700, [700], seed=32)
    q = case.queries(1)
    side = torch.cuda.Stream()
    codes, scale, qkv = _dev(case.packed, dev), _dev(case.scale, dev), _qkv(q, dev)
    cur = torch.tensor([699], dtype=torch.int32, device=dev)
    ws = kvattn.Workspace(1, 2, 700)
    out = torch.empty(1, 2, HS, dtype=torch.bfloat16, device=dev)
    torch.cuda.synchronize()
    kvattn.decode(out, qkv, codes, 1, 2, HS, 700, kv_dtype=kv, kv_scale=scale, cur_len=cur, stream=side, **ws.kwargs())
    side.synchronize()
    case.check(out.float().cpu().numpy(), q, [(0, 0, 700)], "side stream")
