"""Verification of drafted tokens against a sequence-by-sequence restatement in 64 bits (kv4ref.verify)."""
import numpy as np
import pytest

import kv4ref

pytestmark = pytest.mark.gpu


def _kv():
    from cuda_gpt2_inference_amd import kvattn
    return kvattn


def _run(dev, p, q, drafts, u, start, V, dtype="f32", offset=0, ws=None):
    """p, q: float32 [rows, row_stride] (bf16-representable for dtype bf16).  -> tokens, counts.
    offset: elements that the probabilities start behind an aligned address."""
    import torch
    kvattn = _kv()
    rows, stride = p.shape
    B = len(start) - 1
    td = torch.float32 if dtype == "f32" else torch.bfloat16

    def put(x):
        if x is None:
            return None
        flat = torch.empty(x.size + offset, dtype=td, device=dev)
        flat[offset:] = torch.from_numpy(np.ascontiguousarray(x)).view(-1).to(td)
        return flat[offset:]
    pd, qd = put(p), put(q)
    i32 = lambda x: torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(dev)   # noqa: E731
    ud = torch.from_numpy(np.ascontiguousarray(u, dtype=np.float32)).to(dev)
    tokens = torch.full((rows + 4,), -2, dtype=torch.int32, device=dev)
    counts = torch.full((B + 2,), -2, dtype=torch.int32, device=dev)
    nbytes = kvattn.verify_workspace_bytes(B, V)
    if ws is None:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        kvattn.workspace_init(ws, nbytes)
    kvattn.verify_drafts(tokens, counts, pd, i32(drafts), ud, i32(start), B, rows, V, draft_probs=qd, row_stride=stride,
                         dtype=dtype, workspace=ws, workspace_nbytes=nbytes)
    tokens, counts = tokens.cpu().numpy(), counts.cpu().numpy()
    assert (tokens[rows:] == -2).all() and (counts[B:] == -2).all()
    return tokens[:rows], counts[:B]


def _case(r, counts, V, stride, dtype, sure, spare=0):
    rows = int(sum(counts)) + spare
    z = 2.5 * r.standard_normal((rows, V))
    zq = z + 0.7 * r.standard_normal((rows, V))
    soft = lambda a: np.exp(a - a.max(-1, keepdims=True)) / np.exp(a - a.max(-1, keepdims=True)).sum(-1, keepdims=True)  # noqa: E731
    p, q = soft(z), soft(zq)
    drafts = np.array([r.choice(V, p=q[i] / q[i].sum()) for i in range(rows)])

    def store(x):
        out = np.full((rows, stride), np.nan, dtype=np.float32)   # what lies behind the vocabulary is not read
        out[:, :V] = x
        if dtype == "bf16":
            import torch
            out = torch.from_numpy(out).to(torch.bfloat16).float().numpy()
        return out
    start = np.concatenate([[0], np.cumsum(counts)])
    return store(p), None if sure else store(q), drafts, r.rand(rows).astype(np.float32), start


def _check(dev, case, V, dtype="f32", **kw):
    p, q, drafts, u, start = case
    with np.errstate(invalid="ignore"):
        want = kv4ref.verify(p.astype(np.float64), None if q is None else q.astype(np.float64), drafts, u, start, V)
    got = _run(dev, p, q, drafts, u, start, V, dtype, **kw)
    assert np.array_equal(got[1], want[1])
    assert np.array_equal(got[0], want[0])
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sure", [False, True])
@pytest.mark.parametrize("counts,V,stride,offset", [
    ([1], 1, 1, 0), ([3], 2, 2, 0), ([5, 0, 1, 8], 255, 256, 0), ([2, 4], 1024, 1024, 0), ([4, 3, 2], 1025, 1028, 0),
    ([4] * 5, 4099, 4099, 0), ([3] * 4, 4099, 4100, 1), ([5], 50257, 50304, 0), ([8] * 9, 50257, 50304, 0),
    ([2] * 300, 700, 701, 3),
])
def test_verify(dev, dtype, sure, counts, V, stride, offset):
    r = np.random.RandomState(V + len(counts))
    _check(dev, _case(r, counts, V, stride, dtype, sure, spare=2), V, dtype, offset=offset)


@pytest.mark.parametrize("sure", [False, True])
def test_many_drafts(dev, sure):
    """More drafts than a wave has lanes; all accepted, or refused late."""
    r = np.random.RandomState(5)
    counts, V = [130, 65, 64, 200], 50
    p, q, drafts, u, start = _case(r, counts, V, V, "f32", sure)
    u[:] = 0.0                                   # accepts whatever the target gives any mass
    u[start[0] + 70], u[start[3] + 128] = 0.9999999, 0.9999999
    p[start[0] + 70, drafts[start[0] + 70]] = 1e-9
    p[start[3] + 128, drafts[start[3] + 128]] = 1e-9
    if q is not None:
        q[:, :] = 0.01
        q[np.arange(len(drafts)), drafts] = 0.51
    got = _check(dev, (p, q, drafts, u, start), V)
    assert list(got[1]) == [71, 65, 64, 129]


def test_borders_are_exact(dev):
    """Dyadic probabilities: the number on a border draws the next token, just below it the one before."""
    V = 3000
    p = np.zeros((1, V), np.float32)
    where = [0, 1, 255, 256, 1023, 1024, 2048, 2999]
    p[0, where] = 0.125
    eps = 2.0 ** -24
    for i in range(8):
        for u, want in ((i / 8, where[i]), (i / 8 + eps * 8, where[i]), ((i + 1) / 8 - eps, where[i])):
            got = _check(dev, (p, None, np.zeros(1), np.array([u]), np.array([0, 1])), V)
            assert got[0][0] == want
    # Accept iff r q < p: equality refuses.
    p2 = np.full((2, 4), 0.25, np.float32)
    q2 = np.array([[0.5, 0.25, 0.125, 0.125]] * 2, np.float32)
    for u, n in ((0.5, 1), (0.5 - eps, 2)):
        got = _check(dev, (p2, q2, np.array([0, 0]), np.array([u, 0.3]), np.array([0, 2])), 4)
        assert got[1][0] == n


def test_numbers_outside_the_unit_interval(dev):
    """A number of one or more draws the last token with any mass, one below zero (or NaN in the
    test of a draft: refused) the first."""
    V = 2500
    p = np.zeros((1, V), np.float32)
    p[0, 7], p[0, 1500], p[0, 2400] = 0.2, 0.5, 0.3
    for u, want in ((1.0, 2400), (5.0, 2400), (-1.0, 7), (np.inf, 2400), (-np.inf, 7)):
        assert _run(dev, p, None, np.zeros(1), np.array([u]), np.array([0, 1]), V)[0][0] == want
    p2 = np.concatenate([p, p])
    tokens, counts = _run(dev, p2, p2, np.array([1500, 0]), np.array([np.nan, 0.5]), np.array([0, 2]), V)
    assert counts[0] == 1 and tokens[0] == 1500      # p = q leaves nothing, so p itself is drawn from


def test_nothing_to_draw_from(dev):
    """p = q at the refusal: p itself; a row without mass draws no token."""
    V = 40
    p = np.zeros((3, V), np.float32)
    q = np.zeros((3, V), np.float32)
    p[0, 3] = p[0, 30] = q[0, 3] = q[0, 30] = 0.5
    tokens, counts = _check(dev, (p, q, np.array([11, 0, 0]), np.array([0.1, 0.2, 0.75]), np.array([0, 3])), V)
    assert counts[0] == 1 and tokens[0] == 30
    p[0] = 0
    tokens, counts = _check(dev, (p, q, np.array([11, 0, 0]), np.array([0.1, 0.2, 0.75]), np.array([0, 3])), V)
    assert counts[0] == 0 and (tokens == -1).all()
    # A sure draft that was all of p.
    p[0, 5] = 1.0
    tokens, counts = _run(dev, p[:2], None, np.array([5, 0]), np.array([1.0, 0.5]), np.array([0, 2]), V)
    assert counts[0] == 1 and tokens[0] == 5


def test_strange_probabilities_and_drafts(dev):
    """NaN, infinite and negative probabilities weigh nothing; drafts outside the vocabulary are refused."""
    V = 1500
    r = np.random.RandomState(9)
    p = r.rand(6, V).astype(np.float32)
    q = r.rand(6, V).astype(np.float32)
    p[0, 100:110], p[0, 200], p[0, 300:320], q[0, 400:420], q[0, 500] = np.nan, np.inf, -1.0, np.nan, -np.inf
    p[5, ::2] = np.nan
    drafts = np.array([-1, V, 2 ** 31 - 1, 105, 7, 0])
    for start in ([0, 6], [0, 2, 4, 6]):
        _check(dev, (p, q, drafts, r.rand(6).astype(np.float32), np.array(start)), V)
    _check(dev, (p, None, drafts, r.rand(6).astype(np.float32), np.array([0, 2, 4, 6])), V)


def test_wrong_starts_stay_inside(dev):
    V = 64
    r = np.random.RandomState(10)
    p, q, drafts, u, _ = _case(r, [4], V, V, "f32", False)
    got = _run(dev, p, q, drafts, u, np.array([-5, 2, 100, 3]), V)
    want = kv4ref.verify(p.astype(np.float64), q.astype(np.float64), drafts, u, [0, 2, 4], V)
    assert np.array_equal(got[0], want[0]) and list(got[1]) == list(want[1]) + [0]


@pytest.mark.parametrize("counts,V", [([5, 1, 0, 8], 50257), ([4] * 40, 3000), ([100, 3], 200)])
def test_tokens_in_the_drafts_place(dev, counts, V):
    """tokens may be draft_tokens, here on another stream than the default one."""
    import torch
    kvattn = _kv()
    r = np.random.RandomState(14)
    p, q, drafts, u, start = _case(r, counts, V, V, "f32", False, spare=2)
    want = kv4ref.verify(p.astype(np.float64), q.astype(np.float64), drafts, u, start, V)
    t = lambda x, d: torch.from_numpy(np.ascontiguousarray(x)).to(d).to(dev)      # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tokens, counted = t(drafts, torch.int32), torch.zeros(len(counts), dtype=torch.int32, device=dev)
        nbytes = kvattn.verify_workspace_bytes(len(counts), V)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        kvattn.workspace_init(ws, nbytes)
        kvattn.verify_drafts(tokens, counted, t(p, torch.float32), tokens, t(u, torch.float32), t(start, torch.int32), len(counts),
                             len(u), V, draft_probs=t(q, torch.float32), workspace=ws, workspace_nbytes=nbytes)
        got = tokens.cpu().numpy()
    n = int(start[-1])
    assert np.array_equal(got[:n], want[0][:n]) and np.array_equal(got[n:], drafts[n:])
    assert np.array_equal(counted.cpu().numpy(), want[1])


def test_repeats_and_capture(dev):
    """The workspace is left as it was; a captured call replayed on new numbers equals the eager one."""
    import torch
    kvattn = _kv()
    V, B = 5000, 6
    r = np.random.RandomState(11)
    p, q, drafts, u, start = _case(r, [4] * B, V, V, "f32", False)
    t = lambda x, d: torch.from_numpy(np.ascontiguousarray(x)).to(d).to(dev)      # noqa: E731
    pd, qd, dd, sd = t(p, torch.float32), t(q, torch.float32), t(drafts, torch.int32), t(start, torch.int32)
    ud = torch.zeros(len(u), device=dev)
    nbytes = kvattn.verify_workspace_bytes(B, V)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    kvattn.workspace_init(ws, nbytes)
    tokens = torch.zeros(len(u), dtype=torch.int32, device=dev)
    counts = torch.zeros(B, dtype=torch.int32, device=dev)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kvattn.verify_drafts(tokens, counts, pd, dd, ud, sd, B, len(u), V, draft_probs=qd, workspace=ws, workspace_nbytes=nbytes)
    for i in range(5):
        u = r.rand(len(u)).astype(np.float32)
        ud.copy_(t(u, torch.float32))
        graph.replay()
        torch.cuda.synchronize()
        want = kv4ref.verify(p.astype(np.float64), q.astype(np.float64), drafts, u, start, V)
        assert np.array_equal(tokens.cpu().numpy(), want[0]) and np.array_equal(counts.cpu().numpy(), want[1])
        assert not ws[:256].any()


@pytest.mark.parametrize("B,V", [(1, 100), (5, 50257), (600, 9000)])
def test_batch_without_tokens(dev, B, V):
    """Arrays of no elements (their address is none): every count is zero."""
    p = np.zeros((0, V), np.float32)
    for q in (p, None):
        tokens, counts = _run(dev, p, q, np.zeros(0), np.zeros(0), np.zeros(B + 1), V)
        assert tokens.size == 0 and not counts.any()


def test_one_workspace_for_batches_of_every_size(dev):
    """One buffer, zeroed once and sized for the largest, serves calls of any B and V in any order: what one
    leaves in it is no other's business (V from 8193 on takes several workgroups a sequence)."""
    import torch
    kvattn = _kv()
    calls = [(64, 50257), (96, 20000), (300, 9000), (500, 8200), (5, 50257), (1, 100000), (64, 300), (129, 8193), (513, 9000),
             (2, 70000), (96, 20000)]
    nbytes = max(kvattn.verify_workspace_bytes(B, V) for B, V in calls)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    kvattn.workspace_init(ws, nbytes)
    r = np.random.RandomState(21)
    for B, V in calls:
        counts = np.where(np.arange(B) % 3 == 0, 2, 1)
        counts[B // 2] = B > 1 and V % 2                  # one without tokens
        case = _case(r, counts, V, V, "f32", B % 2 == 0)
        _check(dev, case, V, ws=ws)
        assert not ws.any(), (B, V)


def test_two_captured_calls_share_a_workspace(dev):
    """Graphs of different batches over one workspace, replayed in turn."""
    import torch
    kvattn = _kv()
    r = np.random.RandomState(22)
    t = lambda x, d: torch.from_numpy(np.ascontiguousarray(x)).to(d).to(dev)      # noqa: E731
    shapes = [(64, 20000), (80, 16400)]
    nbytes = max(kvattn.verify_workspace_bytes(B, V) for B, V in shapes)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    kvattn.workspace_init(ws, nbytes)
    held = []
    for B, V in shapes:
        p, q, drafts, u, start = _case(r, [2] * B, V, V, "f32", False)
        d = dict(p=t(p, torch.float32), q=t(q, torch.float32), drafts=t(drafts, torch.int32), u=t(u, torch.float32),
                 start=t(start, torch.int32), tokens=torch.full((2 * B,), -2, dtype=torch.int32, device=dev),
                 counts=torch.full((B,), -2, dtype=torch.int32, device=dev), host=(p, q, drafts, start, V))
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            kvattn.verify_drafts(d["tokens"], d["counts"], d["p"], d["drafts"], d["u"], d["start"], B, 2 * B, V,
                                 draft_probs=d["q"], workspace=ws, workspace_nbytes=nbytes)
        held.append((graph, d))
    for i in range(3):
        for graph, d in held:
            u = r.rand(d["u"].numel()).astype(np.float32)
            d["u"].copy_(t(u, torch.float32))
            d["tokens"].fill_(-2)
            d["counts"].fill_(-2)
            graph.replay()
            torch.cuda.synchronize()
            p, q, drafts, start, V = d["host"]
            want = kv4ref.verify(p.astype(np.float64), q.astype(np.float64), drafts, u, start, V)
            assert np.array_equal(d["tokens"].cpu().numpy(), want[0]) and np.array_equal(d["counts"].cpu().numpy(), want[1])
