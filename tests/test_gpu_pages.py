"""Block tables and slot maps from request lengths, and cache rows by slot map, against a
request-by-request restatement (kv4ref.Pool) and the one-token append."""
import numpy as np
import pytest

import kv4ref
from kv4ref import HS

pytestmark = pytest.mark.gpu


def _kv():
    from cuda_gpt2_inference_amd import kvattn
    return kvattn


def _i32(x, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(dev)


class Requests:
    """A paged cache's tables on the device beside the restatement's."""

    def __init__(self, dev, B, n, R, P, head=0):
        import torch
        kvattn = _kv()
        self.dev, self.B, self.n, self.R, self.P = dev, B, n, R, P
        self.table = np.full((B, n), -7, np.int32)
        self.d_table = _i32(self.table, dev)
        self.cache = kvattn.PagedCache(None, self.d_table, n, R, P)
        self.pool = kvattn.paged_pool(P, device=dev)
        assert self.pool.tolist() == [0, P, 0, 0] + list(range(P))
        self.model = kv4ref.Pool(P)
        self.d_held = torch.zeros(B, dtype=torch.int32, device=dev)
        self.held = np.zeros(B, np.int64)

    def step(self, kept, fresh, most, in_place=True, positions=True):
        import torch
        kvattn = _kv()
        B = self.B
        kept_d = _i32(kept, self.dev)
        lens = kept_d if in_place else torch.full((B,), -9, dtype=torch.int32, device=self.dev)
        start = torch.full((B + 1,), -9, dtype=torch.int32, device=self.dev)
        slots = torch.full((max(most, 1) + 5,), -9, dtype=torch.int64, device=self.dev)
        pos = torch.full((max(most, 1) + 5,), -9, dtype=torch.int32, device=self.dev)
        held_out = None if in_place else torch.full((B,), -9, dtype=torch.int32, device=self.dev)
        nxt = None if in_place else torch.full((2,), -9, dtype=torch.int32, device=self.dev)
        before = self.pool.clone()
        kvattn.paged_reserve(self.cache, self.pool, self.d_held, kept_d, _i32(fresh, self.dev), B, held_out=held_out,
                             lens=lens, token_start=start, slot_map=slots, max_tokens=most,
                             positions=pos if positions else None, pool_next=nxt)
        if not in_place:
            assert torch.equal(self.pool[:4], before[:4])
            self.pool[:2] = nxt
            self.d_held = held_out
        w = self.model.reserve(self.table, self.R, self.held, kept, fresh, most)
        self.held = w[0]
        assert np.array_equal(self.d_table.cpu().numpy(), self.table)
        assert self.pool[:4].tolist() == [self.model.head, self.model.count, 0, 0]
        assert np.array_equal(self.pool[4:].cpu().numpy(), self.model.ring)
        assert np.array_equal(self.d_held.cpu().numpy(), w[0])
        assert np.array_equal(lens.cpu().numpy(), w[1])
        assert np.array_equal(start.cpu().numpy(), w[2])
        got, k = slots.cpu().numpy(), len(w[3])
        assert np.array_equal(got[:k], w[3]) and (got[k:most] == -1).all() and (got[max(most, k):] == -9).all()
        got = pos.cpu().numpy()
        if positions:
            assert np.array_equal(got[:k], w[4]) and (got[k:] == -9).all()
        else:
            assert (got == -9).all()
        return w


@pytest.mark.parametrize("B,n,R,P,top,most", [
    (1, 1, 1, 1, 1, 1), (1, 8, 64, 8, 300, 300), (5, 4, 64, 12, 90, 200), (64, 16, 64, 300, 8, 512),
    (65, 16, 64, 300, 8, 512), (200, 8, 64, 400, 6, 1000),
    (257, 12, 96, 900, 400, 30000), (1000, 33, 64, 9000, 300, 200000), (4096, 4, 128, 5000, 200, 100000),
])
@pytest.mark.parametrize("in_place", [True, False])
def test_reserve(dev, B, n, R, P, top, most, in_place):
    """Steps of growth, refused drafts, ends and shortage; the ring goes round."""
    r = np.random.RandomState(B + P)
    rq = Requests(dev, B, n, R, P)
    for i in range(8):
        ends = r.rand(B) < 0.15
        kept = np.where(ends, 0, rq.held - np.minimum(rq.held, r.randint(0, 2 * R, B) * (r.rand(B) < 0.4)))
        fresh = np.minimum(r.randint(0, top + 1, B) * (r.rand(B) < 0.8), n * R - kept)
        fresh = np.where(ends & (r.rand(B) < 0.5), 0, fresh)
        rq.step(kept, fresh, most, in_place, positions=i % 2 == 0)


def test_reserve_refuses_senseless_lengths(dev):
    rq = Requests(dev, 9, 4, 64, 20)
    rq.step(np.zeros(9, np.int64), np.full(9, 70), 1000)
    held = rq.held.copy()
    kept = np.array([-1, 71, 70, 70, 70, 0, 70, -2 ** 31, 2 ** 31 - 1])
    fresh = np.array([5, 5, -1, 187, 186, 256, 2 ** 31 - 1, 3, 2 ** 31 - 1])
    w = rq.step(kept, fresh, 1000)
    assert list(w[0][[0, 1, 2, 3, 6, 7, 8]]) == list(held[[0, 1, 2, 3, 6, 7, 8]])
    assert w[2][-1] == 186 + 256
    # What a request holds may be senseless too.
    rq2 = Requests(dev, 3, 4, 64, 20)
    rq2.held = np.array([-5, 257, 0])
    rq2.d_held = _i32(rq2.held, dev)
    rq2.step(np.array([0, 0, 0]), np.array([1, 1, 1]), 10)


def test_reserve_shortage_of_tokens_and_pages(dev):
    """First come, first served; requests that need no page are still granted."""
    rq = Requests(dev, 6, 4, 64, 5)
    w = rq.step(np.zeros(6, np.int64), np.array([64, 128, 65, 0, 64, 64]), 1000)      # 5 pages: 1, 2, 2, -, none left
    assert list(w[0]) == [64, 128, 65, 0, 0, 0] and (w[3][-128:] == -1).all()
    w = rq.step(np.array([63, 0, 65, 0, 0, 0]), np.array([1, 0, 2, 0, 1, 0]), 2)      # request 2's tokens end behind 2
    assert list(w[0]) == [64, 0, 65, 0, 0, 0]
    w = rq.step(np.array([64, 0, 65, 0, 0, 0]), np.array([0, 0, 1, 64, 64, 64]), 1000)  # the two given back
    assert list(w[0]) == [64, 0, 66, 64, 64, 0]
    w = rq.step(np.zeros(6, np.int64), np.zeros(6, np.int64), 0)
    assert rq.model.count == 5


def test_reserve_sums_past_31_bits(dev):
    """More tokens and pages asked for than an int holds."""
    import torch
    B, n, R, P = 600, 1 << 17, 64, 40
    kvattn = _kv()
    table = torch.full((B, n), -1, dtype=torch.int32, device=dev)
    cache = kvattn.PagedCache(None, table, n, R, P)
    pool = kvattn.paged_pool(P, device=dev)
    held = torch.zeros(B, dtype=torch.int32, device=dev)
    fresh = torch.full((B,), n * R, dtype=torch.int32, device=dev)
    fresh[0] = 100
    kept, lens, start = held.clone(), held.clone(), torch.empty(B + 1, dtype=torch.int32, device=dev)
    slots = torch.full((500,), -9, dtype=torch.int64, device=dev)
    kvattn.paged_reserve(cache, pool, held, kept, fresh, B, lens=lens, token_start=start, slot_map=slots, max_tokens=500)
    assert held.tolist() == [100] + [0] * (B - 1) and lens.tolist() == held.tolist()
    assert slots.tolist() == list(range(100)) + [-1] * 400
    assert start[:3].tolist() == [0, 100, 100 + n * R] and int(start[-1]) == 2 ** 31 - 1
    assert pool[:4].tolist() == [2, 38, 0, 0]


def test_reserve_foreign_pool_stays_inside(dev):
    """Counts and heads that no call of ours left: nothing outside table, ring and outputs is touched."""
    import torch
    kvattn = _kv()
    for head, count in [(-3, 2), (10 ** 9, 99), (2, -4), (-2 ** 31, 2 ** 31 - 1)]:
        guard = torch.full((4 + 8 + 50,), 77, dtype=torch.int32, device=dev)
        guard[:12] = torch.tensor([head, count, 0, 0] + list(range(8)))
        table = torch.full((3, 4), 5, dtype=torch.int32, device=dev)
        cache = kvattn.PagedCache(None, table, 4, 64, 8)
        held = torch.tensor([200, 0, 64], dtype=torch.int32, device=dev)
        kept = torch.tensor([0, 0, 64], dtype=torch.int32, device=dev)
        fresh = torch.tensor([0, 100, 64], dtype=torch.int32, device=dev)
        lens, start = kept.clone(), torch.empty(4, dtype=torch.int32, device=dev)
        slots = torch.full((164,), -9, dtype=torch.int64, device=dev)
        kvattn.paged_reserve(cache, guard, held, kept, fresh, 3, lens=lens, token_start=start, slot_map=slots,
                             max_tokens=164)
        assert (guard[12:] == 77).all() and 0 <= int(guard[0]) < 8 and 0 <= int(guard[1]) <= 8
        assert (slots < 8 * 64).all()


def test_reserve_captured(dev):
    """Allocation inside a captured step: replays go on from the pool the last one left."""
    import torch
    kvattn = _kv()
    B, n, R, P = 3, 4, 64, 9
    rq = Requests(dev, B, n, R, P)
    kept, fresh = torch.zeros(B, dtype=torch.int32, device=dev), torch.zeros(B, dtype=torch.int32, device=dev)
    lens, start = torch.zeros(B, dtype=torch.int32, device=dev), torch.zeros(B + 1, dtype=torch.int32, device=dev)
    slots = torch.zeros(300, dtype=torch.int64, device=dev)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kvattn.paged_reserve(rq.cache, rq.pool, rq.d_held, kept, fresh, B, lens=lens, token_start=start, slot_map=slots,
                             max_tokens=300)
    for i in range(7):
        k = np.where(np.arange(B) == i % B, 0, rq.held)
        f = np.minimum([50, 70, 20], n * R - k)
        kept.copy_(_i32(k, dev))
        fresh.copy_(_i32(f, dev))
        graph.replay()
        torch.cuda.synchronize()
        w = rq.model.reserve(rq.table, R, rq.held, k, f, 300)
        rq.held = w[0]
        assert np.array_equal(rq.d_table.cpu().numpy(), rq.table) and np.array_equal(rq.d_held.cpu().numpy(), w[0])
        assert rq.pool[:4].tolist() == [rq.model.head, rq.model.count, 0, 0]
        assert np.array_equal(slots[:len(w[3])].cpu().numpy(), w[3])
        torch.zeros(1000, device=dev).sum().item()


def test_reserve_captured_many_requests(dev):
    """A captured call whose requests need more LDS than a launch gets by itself, replayed in place."""
    import torch
    kvattn = _kv()
    B, n, R, P, most = 3500, 2, 64, 6000, 40000
    r = np.random.RandomState(4)
    rq = Requests(dev, B, n, R, P)
    z = lambda k, t=torch.int32: torch.zeros(k, dtype=t, device=dev)         # noqa: E731
    kept, fresh, lens, start, slots = z(B), z(B), z(B), z(B + 1), z(most, torch.int64)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kvattn.paged_reserve(rq.cache, rq.pool, rq.d_held, kept, fresh, B, lens=lens, token_start=start, slot_map=slots,
                             max_tokens=most)
    for i in range(4):
        k = np.where(r.rand(B) < 0.3, 0, rq.held)
        f = np.minimum(r.randint(0, 20, B), n * R - k)
        kept.copy_(_i32(k, dev))
        fresh.copy_(_i32(f, dev))
        graph.replay()
        torch.cuda.synchronize()
        w = rq.model.reserve(rq.table, R, rq.held, k, f, most)
        rq.held = w[0]
        assert np.array_equal(rq.d_table.cpu().numpy(), rq.table) and np.array_equal(rq.d_held.cpu().numpy(), w[0])
        assert np.array_equal(lens.cpu().numpy(), w[1]) and np.array_equal(start.cpu().numpy(), w[2])
        assert rq.pool[:4].tolist() == [rq.model.head, rq.model.count, 0, 0]
        assert np.array_equal(slots[:len(w[3])].cpu().numpy(), w[3]) and (slots[len(w[3]):] == -1).all()


# ------------------------------------------------------------------------------------
# Rows by slot.
# ------------------------------------------------------------------------------------
def _pool(kv, P, NH, R, dev):
    import torch
    store = {"f32": torch.float32, "bf16": torch.bfloat16}.get(kv, torch.uint8)
    width = HS // 2 if kv in ("int4", "fp4") else HS
    fill = 9 if store == torch.uint8 else 9.0
    pages = torch.full((P, 2, NH, R, width), fill, dtype=store, device=dev)
    scales = None if kv in ("f32", "bf16") else torch.full((P, 2, NH, R), -5.0, device=dev)
    return pages, scales


@pytest.mark.parametrize("kv", ["f32", "bf16", "int8", "fp8", "int4", "fp4"])
@pytest.mark.parametrize("n,NH,R", [(1, 1, 1), (7, 3, 64), (8, 12, 64), (65, 5, 96), (1000, 2, 128)])
def test_store_is_the_append(dev, kv, n, NH, R):
    """Rows by slot equal the one-token append's, bit for bit, and nothing else changes; slots outside the
    pool are skipped.  Loaded rows are code times scale."""
    import torch
    kvattn = _kv()
    P = -(-n // R) + 2
    act = torch.float32 if kv == "f32" else torch.bfloat16
    g = torch.Generator().manual_seed(n + NH)
    qkv = (torch.randn(n, 3, NH, HS, generator=g) * 10 ** torch.randn(n, 3, NH, 1, generator=g)).to(act).to(dev)
    if n > 5:
        qkv[2, 1:] = 0
        qkv[3, 1, 0, 5] = float("inf")
    slots = torch.randperm(P * R, generator=g)[:n]
    if n > 5:
        slots[1], slots[4], slots[5] = -1, P * R, 2 ** 62
    slots_d = slots.to(dev)
    pages, scales = _pool(kv, P, NH, R, dev)
    cache = kvattn.PagedCache(pages, None, 1, R, P, scales)
    kvattn.paged_store(cache, qkv, slots_d, n, NH, HS, kv_dtype=kv)
    # One sequence a token, contiguous, position 0.
    one = torch.zeros((2, n, NH, 1) + pages.shape[-1:], dtype=pages.dtype, device=dev)
    one_s = None if scales is None else torch.zeros(2, n, NH, 1, device=dev)
    kvattn.kv_cache_write(one, qkv, n, NH, HS, 1, kv_dtype=kv, kv_scale=one_s,
                          cur_len=torch.zeros(1, dtype=torch.int32, device=dev))
    want, want_s = _pool(kv, P, NH, R, dev)
    live = ((slots >= 0) & (slots < P * R)).nonzero().view(-1)
    page, row = (slots[live] // R).to(dev), (slots[live] % R).to(dev)
    want[page, :, :, row] = one[:, live.to(dev), :, 0].transpose(0, 1)
    as_int = lambda t: t.view({4: torch.int32, 2: torch.int16, 1: torch.uint8}[t.element_size()])   # noqa: E731
    assert torch.equal(as_int(pages), as_int(want))
    if scales is not None:
        want_s[page, :, :, row] = one_s[:, live.to(dev), :, 0].transpose(0, 1)
        assert torch.equal(as_int(scales), as_int(want_s))
    back = torch.full((n, 2, NH, HS), 3.0, dtype=act, device=dev)
    kvattn.paged_load(back, cache, slots_d, n, NH, HS, kv_dtype=kv)
    ref = torch.full((n, 2, NH, HS), 3.0, dtype=act)
    rows = pages[page, :, :, row].cpu()
    if kv in ("f32", "bf16"):
        vals = rows
    else:
        sc = scales[page, :, :, row].cpu()
        if kv == "int8":
            code = rows.view(torch.int8).float()
        elif kv == "fp8":
            code = rows.view(torch.float8_e4m3fn).float()
        else:
            code = torch.from_numpy(kv4ref.decode(rows.numpy(), np.ones(sc.shape), kv)).float()
        vals = (code * sc.unsqueeze(-1)).to(act)
    ref[live] = vals
    same = (as_int(back.cpu()) == as_int(ref)) | (torch.isnan(back.cpu().float()) & torch.isnan(ref.float()))
    assert same.all()


@pytest.mark.parametrize("kv", ["int4", "fp8"])
def test_rows_captured(dev, kv):
    import torch
    kvattn = _kv()
    n, NH, R, P = 33, 2, 64, 4
    pages, scales = _pool(kv, P, NH, R, dev)
    cache = kvattn.PagedCache(pages, None, 1, R, P, scales)
    qkv = torch.zeros(n, 3, NH, HS, dtype=torch.bfloat16, device=dev)
    slots = torch.zeros(n, dtype=torch.int64, device=dev)
    back = torch.zeros(n, 2, NH, HS, dtype=torch.bfloat16, device=dev)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kvattn.paged_store(cache, qkv, slots, n, NH, HS, kv_dtype=kv)
        kvattn.paged_load(back, cache, slots, n, NH, HS, kv_dtype=kv)
    for i in range(4):
        g = torch.Generator().manual_seed(i)
        qkv.copy_(torch.randn(n, 3, NH, HS, generator=g))
        slots.copy_(torch.randperm(P * R, generator=g)[:n])
        graph.replay()
        torch.cuda.synchronize()
        p2, s2 = _pool(kv, P, NH, R, dev)
        b2 = torch.zeros_like(back)
        c2 = kvattn.PagedCache(p2, None, 1, R, P, s2)
        kvattn.paged_store(c2, qkv, slots, n, NH, HS, kv_dtype=kv)
        kvattn.paged_load(b2, c2, slots, n, NH, HS, kv_dtype=kv)
        assert torch.equal(b2, back)


@pytest.mark.parametrize("kv", ["int4", "fp4"])
def test_every_quotient_rounds_as_the_division(dev, kv):
    """Codes of every pair of bf16 significands (a row's largest element and another) whose quotient can
    reach a code of its own, in the middle of the range and at its ends: bit for bit the definition's."""
    import torch
    kvattn = _kv()
    sig = 1 + np.arange(128) / 128.0
    others = (sig[None, :] * 2.0 ** -np.arange(6)[:, None]).reshape(-1)       # 768 magnitudes, 1 .. 2^-5
    rows = np.zeros((128, 13, 64), np.float32)
    flat = np.concatenate([others, -others[:51]])                             # 13 * 63 = 819
    rows[:, :, 1:] = flat.reshape(1, 13, 63)
    rows[:, :, 0] = 2 * sig[:, None]                                          # the largest
    for shift in (0, 80, -85, 118, -110):
        x = (rows * np.float32(2.0) ** shift).reshape(-1, 64)
        qkv = torch.zeros(x.shape[0], 3, 1, HS, dtype=torch.bfloat16, device=dev)
        qkv[:, 1, 0] = torch.from_numpy(x).to(torch.bfloat16).to(dev)
        n = x.shape[0]
        pages, scales = _pool(kv, 1, 1, n, dev)
        cache = kvattn.PagedCache(pages, None, 1, n, 1, scales)
        kvattn.paged_store(cache, qkv, torch.arange(n, device=dev), n, 1, HS, kv_dtype=kv)
        want, want_s = kv4ref.encode(qkv[:, 1, 0].float().cpu().numpy(), kv)
        assert np.array_equal(scales[0, 0, 0].cpu().numpy(), want_s)
        assert np.array_equal(pages[0, 0, 0].cpu().numpy(), want)


@pytest.mark.parametrize("kv", ["int4", "fp4"])
@pytest.mark.parametrize("beside", ["plain", "zeros", "nan"])
def test_negative_zero_keeps_its_code(dev, kv, beside):
    """-0 (and a negative value that rounds to no magnitude) has the code that the definition gives it, whatever rows
    its wave's other tokens are."""
    import torch
    kvattn = _kv()
    r = np.random.RandomState(3)
    x = r.standard_normal((8, HS)).astype(np.float32)
    x[:, ::3] = -0.0
    x[:, 1::7] = 0.0
    x[:, 2::9] = -1e-6
    if beside == "zeros":
        x[3] = 0.0
    elif beside == "nan":
        x[3, 5] = np.nan
    qkv = torch.zeros(8, 3, 1, HS, dtype=torch.bfloat16, device=dev)
    qkv[:, 1, 0] = torch.from_numpy(x).to(torch.bfloat16).to(dev)
    pages, scales = _pool(kv, 1, 1, 64, dev)
    kvattn.paged_store(kvattn.PagedCache(pages, None, 1, 64, 1, scales), qkv, torch.arange(8, device=dev), 8, 1, HS, kv_dtype=kv)
    want, want_s = kv4ref.encode(qkv[:, 1, 0].float().cpu().numpy(), kv)
    assert np.array_equal(scales[0, 0, 0, :8].cpu().numpy(), want_s)
    assert np.array_equal(pages[0, 0, 0, :8].cpu().numpy(), want)
