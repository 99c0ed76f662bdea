"""Refusals of the 4-bit cache, paging and draft verification calls (before anything reaches a GPU), the
4-bit plan, and the restatements that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import kv4ref

A = 1 << 20   # a fake aligned address; never dereferenced by these calls
BIG = 1 << 30


def _kv():
    from cuda_gpt2_inference_amd import kvattn
    return kvattn


def _status(entry, args, kw):
    unknown = set(kw) - set(args)
    assert not unknown, unknown
    L = _kv().lib()
    return getattr(L, entry)(*{**args, **kw}.values())


TOKENS = dict(out=A, qkv=A, pages=A, scales=A, table=A, max_pages=4, page_rows=64, num_pages=8, start=A, lens=A, B=2,
              n=5, max_new=3, NH=12, hs=64, ws=A, wsb=BIG, S=0, dt=5, stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(hs=32), 3), (dict(dt=1), 5), (dict(dt=3), 5), (dict(dt=6), 5), (dict(scales=None), 5), (dict(out=None), 1),
    (dict(qkv=None), 1), (dict(pages=None), 1), (dict(table=None), 1), (dict(start=None), 1), (dict(lens=None), 1),
    (dict(out=A + 8), 2), (dict(start=A + 2), 2), (dict(table=A + 1), 2), (dict(scales=A + 2), 2), (dict(ws=A + 4, S=4), 2),
    (dict(B=0), 4), (dict(n=0), 4), (dict(max_new=0), 4), (dict(page_rows=48), 4), (dict(page_rows=96), 4),
    (dict(num_pages=0), 4), (dict(max_pages=1 << 20), 4), (dict(NH=1 << 23), 4), (dict(S=1 << 20), 8), (dict(S=-100), 8),
    (dict(ws=None, S=4), 7), (dict(wsb=1000, S=4), 7), (dict(wsb=0, S=4), 7),
])
def test_decode_tokens_refusals(kw, status):
    assert _status("kvattn_paged_decode_tokens", TOKENS, kw) == status


@pytest.mark.parametrize("B,n,NH", [(1024, 8192, 12), (4096, 16384, 12), (65535, 1 << 18, 25), (1, 1 << 20, 12)])
@pytest.mark.parametrize("max_new", [9, 64, 8192, 2 ** 31 - 1])
def test_decode_tokens_takes_any_max_new(B, n, NH, max_new):
    """The number of tokens bounds the grid; refused here for the missing workspace of two segments alone."""
    assert _status("kvattn_paged_decode_tokens", TOKENS, dict(B=B, n=n, NH=NH, max_new=max_new, S=2, ws=None)) == 7


@pytest.mark.parametrize("B,NH,n,max_new", [(342, 12, 400, 8), (342, 12, 400, 1), (4096, 12, 8192, 100), (4096, 12, 4096, 2)])
def test_widest_tables_are_taken(B, NH, n, max_new):
    """Tables of 2^23 positions a sequence: the segments that the library picks fit a grid (refused here for the missing
    workspace alone)."""
    kw = dict(B=B, NH=NH, n=n, max_new=max_new, max_pages=1 << 17, ws=None)
    assert _status("kvattn_paged_decode_tokens", TOKENS, kw) == 7


DECODE = dict(out=A, qkv=A, kv=A, scale=A, B=1, NH=12, hs=64, maxT=4096, cur=A, per_seq=0, hint=-1, ws=None, wsb=0, S=4,
              strategy=0, dt=4, stream=None)


@pytest.mark.parametrize("entry", ["kvattn_decode", "kvattn_append_decode"])
@pytest.mark.parametrize("kw,status", [
    (dict(hs=128), 3), (dict(scale=None), 5), (dict(scale=A + 2), 2), (dict(kv=A + 8), 2), (dict(out=None), 1),
    (dict(maxT=0), 4), (dict(strategy=1), 6), (dict(strategy=6), 6), (dict(strategy=9), 6), (dict(hint=4096), 12), ({}, 7),
    (dict(ws=A, wsb=4096), 7), (dict(S=-65), 8),
])
@pytest.mark.parametrize("dt", [4, 5])
def test_decode4_refusals(entry, kw, status, dt):
    assert _status(entry, DECODE, {**kw, "dt": dt}) == status


def test_other_calls_refuse_4bit():
    """What is not documented for 4-bit caches says so."""
    L, kv = _kv().lib(), _kv()
    for dt in (4, 5):
        assert L.kvattn_forward_small(A, A, A, A, 1, 12, 64, 1024, A, 0, dt, None) == kv.ERR_DTYPE
        assert L.kvattn_forward_large(A, A, A, A, 1, 12, 64, 1024, A, 0, A, A, A, 8, dt, None) == kv.ERR_DTYPE
        assert L.kvattn_split(A, A, A, A, A, A, 1, 12, 64, 1024, A, 0, 8, dt, None) == kv.ERR_DTYPE
        assert L.kvattn_decode_static(A, A, A, A, 1, 12, 64, 1024, A, 0, -1, 0, 0, dt, None) == kv.ERR_DTYPE
        assert L.kvattn_gemv(A, None, A, A, A, None, 1, 64, 64, dt, 0, None) == kv.ERR_DTYPE
        assert L.kvattn_gemv_qkv_append(A, A, A, A, None, 1, 12, 64, 768, A, A, 64, A, 0, 2, dt, A, BIG, None) == kv.ERR_DTYPE


RESERVE = dict(table=A, max_pages=16, R=64, P=100, pool=A, held=A, kept=A, fresh=A, B=3, most=10, held_out=A, lens=A, start=A,
               slots=A, positions=A, next=A, stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(B=0), 4), (dict(B=4097), 4), (dict(max_pages=0), 4), (dict(R=0), 4), (dict(P=0), 4), (dict(most=-1), 4),
    (dict(max_pages=1 << 20), 4), (dict(P=(1 << 28) + 1), 4), (dict(table=None), 1), (dict(pool=None), 1),
    (dict(held=None), 1), (dict(kept=None), 1), (dict(fresh=None), 1), (dict(held_out=None), 1), (dict(lens=None), 1),
    (dict(start=None), 1), (dict(slots=None), 1), (dict(pool=A + 2), 2), (dict(slots=A + 4), 2), (dict(positions=A + 1), 2),
    (dict(next=A + 3), 2),
])
def test_reserve_refusals(kw, status):
    assert _status("kvattn_paged_reserve", RESERVE, kw) == status


def test_counts_whose_indices_would_overflow():
    """Refused before the GPU: a thread's walk past its last row would leave 31 bits."""
    for n in (2 ** 30 + 1, 2 ** 31 - 1):
        assert _status("kvattn_paged_reserve", RESERVE, dict(most=n)) == 4
        assert _status("kvattn_verify_drafts", VERIFY, dict(n=n)) == 4


def test_rows_of_more_heads_than_a_grid_takes():
    """2^24 heads, as everywhere: few tokens of more would have more threads than a grid counts."""
    order = ("act", "pages", "scales", "R", "P", "slots", "n", "NH", "hs", "dt", "stream")
    for n, NH in ((1, 1 << 25), (4, 1 << 25), (1, 1 << 27), (1, (1 << 24) + 1), (9, 1 << 24)):
        assert _status("kvattn_paged_store", ROWS, dict(n=n, NH=NH)) == 4
        assert _status("kvattn_paged_load", {k: ROWS[k] for k in order}, dict(n=n, NH=NH)) == 4


def test_pool_calls():
    kv = _kv()
    L = kv.lib()
    assert L.kvattn_paged_pool_bytes(10) == 56
    assert L.kvattn_paged_pool_bytes(0) == 0 and L.kvattn_paged_pool_bytes((1 << 28) + 1) == 0
    assert L.kvattn_paged_pool_init(None, 4, None) == kv.ERR_NULL_POINTER
    assert L.kvattn_paged_pool_init(A + 2, 4, None) == kv.ERR_MISALIGNED
    assert L.kvattn_paged_pool_init(A, 0, None) == kv.ERR_SHAPE


ROWS = dict(pages=A, scales=A, R=64, P=4, slots=A, act=A, n=3, NH=12, hs=64, dt=4, stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(hs=63), 3), (dict(n=0), 4), (dict(NH=0), 4), (dict(R=0), 4), (dict(P=0), 4), (dict(n=1 << 28, NH=64), 4),
    (dict(dt=6), 5), (dict(dt=-1), 5), (dict(scales=None), 5), (dict(scales=None, dt=2), 5), (dict(pages=None), 1),
    (dict(slots=None), 1), (dict(act=None), 1), (dict(act=A + 8), 2), (dict(pages=A + 4), 2), (dict(slots=A + 4), 2),
])
def test_rows_refusals(kw, status):
    assert _status("kvattn_paged_store", ROWS, kw) == status
    order = ("act", "pages", "scales", "R", "P", "slots", "n", "NH", "hs", "dt", "stream")
    assert _status("kvattn_paged_load", {k: ROWS[k] for k in order}, kw) == status


VERIFY = dict(tokens=A, counts=A, p=A, q=A, drafts=A, u=A, start=A, B=2, n=8, V=100, row=100, dt=0, ws=A, wsb=BIG,
              stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(dt=2), 5), (dict(dt=4), 5), (dict(B=0), 4), (dict(B=1 << 17), 4), (dict(V=0), 4), (dict(V=(1 << 24) + 1, row=BIG), 4),
    (dict(row=99), 4), (dict(n=-1), 4), (dict(tokens=None), 1), (dict(counts=None), 1), (dict(p=None), 1),
    (dict(drafts=None), 1), (dict(u=None), 1), (dict(start=None), 1), (dict(p=A + 2), 2), (dict(q=A + 1), 2),
    (dict(p=A + 1, dt=1), 2), (dict(u=A + 2), 2), (dict(ws=A + 16), 2), (dict(ws=None), 7), (dict(wsb=256), 7),
])
def test_verify_refusals(kw, status):
    assert _status("kvattn_verify_drafts", VERIFY, kw) == status


def test_verify_of_no_tokens_needs_no_arrays_of_them():
    none = dict(tokens=None, p=None, q=None, drafts=None, u=None, ws=None)     # refused for its workspace alone
    assert _status("kvattn_verify_drafts", VERIFY, {**none, "n": 0}) == 7
    assert _status("kvattn_verify_drafts", VERIFY, {**none, "n": 1}) == 1
    assert _status("kvattn_verify_drafts", VERIFY, {**none, "n": 0, "counts": None}) == 1
    assert _status("kvattn_verify_drafts", VERIFY, {**none, "n": 0, "start": None}) == 1


def test_verify_workspace_bytes():
    kv = _kv()
    assert kv.verify_workspace_bytes(1, 1) == 512
    assert kv.verify_workspace_bytes(64, 50257) == 256 + 64 * 50 * 16
    assert kv.verify_workspace_bytes(0, 10) == 0 and kv.verify_workspace_bytes(1, 1 << 25) == 0


@pytest.mark.parametrize("dt", ["int4", "fp4"])
def test_plan4(dt):
    kv = _kv()
    for B, NH, maxT, hint in [(1, 12, 1024, -1), (1, 12, 1024, 99), (64, 12, 8192, -1), (1, 1, 1, -1), (3, 25, 100000, -1),
                              (4096, 25, 1 << 23, -1)]:
        st, seg, rows = kv.plan(B, NH, 64, maxT, kv_dtype=dt, len_hint=hint)
        assert st == kv.SPLIT_LASTBLOCK and seg >= 1 and rows % 64 == 0 and rows >= 64
        assert kv.workspace_bytes(B, NH, 64, maxT, seg) > 0
        assert seg <= -(-maxT // 64), "a workspace sized for every choice (S = 0) holds it"
    assert kv.plan(1, 12, 64, 1024, kv_dtype=dt, S=5) == (kv.SPLIT_LASTBLOCK, 5, 0)
    assert kv.plan(1, 12, 64, 1000, kv_dtype=dt, S=-128) == (kv.SPLIT_LASTBLOCK, 8, 128)
    n = ctypes.c_int()
    bad = _kv().lib().kvattn_plan(1, 12, 64, 1024, -1, 0, 1, kv.kv_dtype_code(dt), ctypes.byref(n), ctypes.byref(n),
                                  ctypes.byref(n))
    assert bad == kv.ERR_STRATEGY


# ------------------------------------------------------------------------------------
# The restatements against facts of their own.
# ------------------------------------------------------------------------------------
def test_codes_are_the_nearest():
    r = np.random.RandomState(0)
    x = r.standard_normal((200, 64)).astype(np.float32)
    for kv, grid in (("int4", np.arange(-7, 8.0)), ("fp4", np.concatenate([kv4ref.FP4, -kv4ref.FP4]))):
        packed, scale = kv4ref.encode(x, kv)
        val = kv4ref.decode(packed, scale, kv)
        best = np.abs(x[..., None] - grid * scale.astype(np.float64)[:, None, None]).min(-1)
        assert np.abs(np.abs(val - x) - best).max() < 1e-6
    packed, scale = kv4ref.encode(np.zeros((1, 64), np.float32), "int4")
    assert (packed == 0x88).all() and scale[0] == 0


def test_pool_keeps_every_page():
    """Pages are neither lost nor held twice, whatever is granted and refused."""
    r = np.random.RandomState(1)
    B, n, R, P = 9, 6, 64, 25
    table, pool = np.full((B, n), -1, np.int32), kv4ref.Pool(P)
    held = np.zeros(B, np.int64)
    for _ in range(60):
        kept = (held * (r.rand(B) > 0.2) * r.rand(B)).astype(np.int64)
        fresh = np.minimum(r.randint(0, 200, B), n * R - kept)
        held, lens, start, slots, pos = pool.reserve(table, R, held, kept, fresh, 600)
        used = [table[b, i] for b in range(B) for i in range(-(-int(held[b]) // R))]
        free = [pool.ring[(pool.head + i) % P] for i in range(pool.count)]
        assert sorted(used + free) == list(range(P))
        live = slots[slots >= 0]
        assert len(set(live.tolist())) == len(live)


def test_verified_tokens_follow_the_target():
    """Over a grid of random numbers the emitted first token has the target's distribution, as the
    accept / draw rule promises: sum over drafts of q(x) [accept + refuse * draw] = p."""
    V = 5
    p = np.array([0.1, 0.4, 0.05, 0.25, 0.2])
    q = np.array([0.3, 0.2, 0.1, 0.1, 0.3])
    got, N = np.zeros(V), 400
    for x in range(V):
        for i in range(N):
            for j in range(0, N, 20):
                u = np.array([(i + 0.5) / N, (j + 10) / N])
                tok, cnt = kv4ref.verify(np.stack([p, p]), np.stack([q, q]), np.array([x, 0]), u, [0, 2], V)
                got[tok[0]] += q[x] / (N * N / 20)
    assert np.abs(got - p).max() < 0.01


@pytest.mark.parametrize("kv", ["int4", "fp4"])
def test_bound_rejects_mistakes(kv):
    """The bound that the GPU outputs are held to is passed by a float32 evaluation and failed by one with a
    key left out, a scale off by one row, or the softmax scale off."""
    r = np.random.RandomState(3)
    T = 100
    pk, ks = kv4ref.encode(r.standard_normal((T, 64)).astype(np.float32), kv)
    pv, vs = kv4ref.encode(r.standard_normal((T, 64)).astype(np.float32), kv)
    k, v = kv4ref.decode(pk, ks, kv), kv4ref.decode(pv, vs, kv)
    q = r.standard_normal(64)
    ref, wv = kv4ref.attend(q, k, v, T)
    lim = kv4ref.bound(ref, wv, q, ks, vs, kv, T)
    s = (k.astype(np.float32) @ q.astype(np.float32)) / np.float32(8)
    w = np.exp(s - s.max())
    assert (np.abs((w / w.sum()) @ v.astype(np.float32) - ref) <= lim).all()
    assert (np.abs(kv4ref.attend(q, k, v, T - 1)[0] - ref) > lim).any()
    assert (np.abs(kv4ref.attend(q, k, kv4ref.decode(pv, np.roll(vs, 1), kv), T)[0] - ref) > lim).any()
    assert (np.abs(kv4ref.attend(q * 1.01, k, v, T)[0] - ref) > lim).any()
