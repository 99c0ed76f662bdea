"""Decode attention and append over 4-bit caches, contiguous and paged, one and several tokens a
sequence, against 64-bit attention over the stored values (kv4ref.bound)."""
import numpy as np
import pytest

import kv4ref
from kv4ref import HS

pytestmark = pytest.mark.gpu
KV4 = ["int4", "fp4"]


def _kv():
    from cuda_gpt2_inference_amd import kvattn
    return kvattn


def _bf16(x):
    """float32 values that bf16 holds."""
    import torch
    return torch.from_numpy(np.asarray(x, dtype=np.float32)).to(torch.bfloat16).float().numpy()


def _dev(x, dev, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).to(dev)
    return t if dtype is None else t.to(dtype)


def _qkv(q, dev):
    """q [N, NH, 64] as qkv [N, 3, NH, 64] on the device; K and V hold NaN."""
    import torch
    t = torch.full((q.shape[0], 3) + q.shape[1:], float("nan"), dtype=torch.bfloat16, device=dev)
    t[:, 0] = _dev(q, dev, torch.bfloat16)
    return t


class Case:
    """Rows of B sequences of up to maxT positions and NH heads, in 4 bits."""

    def __init__(self, kv, B, NH, maxT, lens, seed=0, sharp=1.0):
        r = np.random.RandomState(seed)
        self.kv, self.B, self.NH, self.maxT, self.lens, self.r = kv, B, NH, maxT, list(lens), r
        rows = r.standard_normal((2, B, NH, maxT, HS)) * np.exp(0.5 * r.standard_normal((2, B, NH, maxT, 1)))
        self.packed, self.scale = kv4ref.encode(_bf16(rows), kv)
        # Rows that no call may read: every code, a scale that is NaN.
        for b, T in enumerate(self.lens):
            self.scale[:, b, :, T:] = np.nan
        self.sharp = sharp

    def queries(self, N):
        return _bf16(self.sharp * self.r.standard_normal((N, self.NH, HS)))

    def check(self, got, q, tokens, what):
        """tokens: (row of got, sequence, rows seen)."""
        for t, b, seen in tokens:
            for h in range(self.NH):
                T = max(seen, 0)
                k, v = (kv4ref.decode(self.packed[i, b, h, :T], self.scale[i, b, h, :T], self.kv) for i in (0, 1))
                ref, wv = kv4ref.attend(q[t, h].astype(np.float64), k, v, seen)
                lim = kv4ref.bound(ref, wv, q[t, h], self.scale[0, b, h], self.scale[1, b, h], self.kv, seen)
                err = np.abs(got[t, h] - ref)
                assert (err <= lim).all(), f"{what}: token {t} sequence {b} head {h} seen {seen}: {err.max()} {lim[err.argmax()]}"

    def paged(self, R, dev, seed=0, spare=2):
        """A PagedCache of the same rows; pages nobody holds are full of NaN scales."""
        import torch
        kvattn = _kv()
        n = self.maxT // R
        P = self.B * n + spare
        table = np.random.RandomState(seed).permutation(P)[:self.B * n].reshape(self.B, n).astype(np.int32)
        pool = np.full((P, 2, self.NH, R, HS // 2), 0xFF, dtype=np.uint8)
        sc = np.full((P, 2, self.NH, R), np.nan, dtype=np.float32)
        for b in range(self.B):
            for i in range(n):
                pool[table[b, i]] = self.packed[:, b, :, i * R:(i + 1) * R]
                sc[table[b, i]] = self.scale[:, b, :, i * R:(i + 1) * R]
        return kvattn.PagedCache(_dev(pool, dev), _dev(table, dev), n, R, P, _dev(sc, dev)), table


def _decode(case, dev, q, hint=-1, S=0, per_seq=True, **kw):
    import torch
    kvattn = _kv()
    out = torch.full((case.B, case.NH, HS), 7.0, dtype=torch.bfloat16, device=dev)
    cur = _dev(np.array(case.lens, dtype=np.int32) - 1, dev)
    ws = kvattn.Workspace(case.B, case.NH, case.maxT, S)
    kvattn.decode(out, _qkv(q, dev), _dev(case.packed, dev), case.B, case.NH, HS, case.maxT, kv_dtype=case.kv,
                  kv_scale=_dev(case.scale, dev), cur_len=cur, lens_per_seq=per_seq, len_hint=hint, S=S, **ws.kwargs(), **kw)
    return out.float().cpu().numpy()


@pytest.mark.parametrize("kv", KV4)
@pytest.mark.parametrize("maxT,T", [(1, 1), (2, 1), (63, 63), (64, 64), (65, 65), (128, 100), (1000, 999), (1024, 1024),
                                    (2048, 1025), (4100, 4097)])
def test_decode_lengths(dev, kv, maxT, T):
    case = Case(kv, 1, 3, maxT, [T], seed=T)
    q = case.queries(1)
    for hint in (-1, T - 1):
        case.check(_decode(case, dev, q, hint), q, [(0, 0, T)], f"hint {hint}")


@pytest.mark.parametrize("kv", KV4)
@pytest.mark.parametrize("S", [1, 2, 3, 7, 64, 200, -64, -192, -1024])
def test_decode_segments(dev, kv, S):
    """Any number of segments, more than there are tiles among them."""
    lens = [1, 64, 65, 700, 1290]
    case = Case(kv, len(lens), 2, 1300, lens, seed=5)
    q = case.queries(len(lens))
    case.check(_decode(case, dev, q, S=S, strategy="lastblock"), q, [(b, b, T) for b, T in enumerate(lens)], f"S {S}")


@pytest.mark.parametrize("kv", KV4)
def test_decode_short_hint(dev, kv):
    """A hint shorter than the sequence only changes the segments."""
    case = Case(kv, 2, 1, 5000, [4999, 10], seed=6)
    q = case.queries(2)
    case.check(_decode(case, dev, q, hint=0), q, [(0, 0, 4999), (1, 1, 10)], "hint 0")


@pytest.mark.parametrize("kv", KV4)
@pytest.mark.parametrize("sharp", [0.0, 0.1, 8.0, 300.0])
def test_decode_sharpness(dev, kv, sharp):
    """From the mean of all rows to one row alone."""
    case = Case(kv, 2, 2, 3000, [3000, 2111], seed=7, sharp=sharp)
    q = case.queries(2)
    case.check(_decode(case, dev, q), q, [(0, 0, 3000), (1, 1, 2111)], f"sharp {sharp}")


@pytest.mark.parametrize("kv", KV4)
def test_largest_score_keeps_its_weight(dev, kv):
    """Scores of 2^40: the row that has the largest gets weight one, two rows alike share it."""
    import torch
    case = Case(kv, 1, 1, 130, [130], seed=8)
    q = case.queries(1)
    q[0, 0] = np.sign(kv4ref.decode(case.packed[0, 0, 0, 77], case.scale[0, 0, 0, 77], kv)) * 2.0 ** 40
    case.packed[0, 0, 0, 3], case.scale[0, 0, 0, 3] = case.packed[0, 0, 0, 77], case.scale[0, 0, 0, 77]
    case.scale[0, 0, 0, [3, 77]] *= 4
    got = _decode(case, dev, q)[0, 0]
    v = kv4ref.decode(case.packed[1, 0, 0], case.scale[1, 0, 0], kv)
    ref = (v[3] + v[77]) / 2
    assert (np.abs(got - ref) <= (2.0 ** -8 + 2.0 ** -13) * (np.abs(v[3]) + np.abs(v[77]))).all()


@pytest.mark.parametrize("kv", KV4)
def test_decode_one_length_and_library_length(dev, kv):
    """One length for the batch; lengths outside the cache are clamped."""
    import torch
    kvattn = _kv()
    case = Case(kv, 3, 2, 200, [150] * 3, seed=9)
    q = case.queries(3)
    case.check(_decode(case, dev, q, per_seq=False), q, [(b, b, 150) for b in range(3)], "one length")
    full = Case(kv, 2, 1, 100, [100, 1], seed=10)
    q = full.queries(2)
    keep, full.lens = full.lens, [10 ** 6, -5]
    got = _decode(full, dev, q)
    full.lens = keep
    full.check(got, q, [(0, 0, 100), (1, 1, 1)], "clamped")
    kvattn.set_cur_len(149)
    try:
        out = torch.empty(3, 2, HS, dtype=torch.bfloat16, device=dev)
        ws = kvattn.Workspace(3, 2, 200)
        q = case.queries(3)
        for per_seq in (False, True):      # the library holds one length, whatever is asked for
            kvattn.decode(out, _qkv(q, dev), _dev(case.packed, dev), 3, 2, HS, 200, kv_dtype=kv,
                          kv_scale=_dev(case.scale, dev), lens_per_seq=per_seq, **ws.kwargs())
            case.check(out.float().cpu().numpy(), q, [(b, b, 150) for b in range(3)], "library length")
    finally:
        kvattn.set_cur_len(0)


@pytest.mark.parametrize("kv", KV4)
@pytest.mark.parametrize("R", [64, 192, 512])
def test_paged_decode(dev, kv, R):
    import torch
    kvattn = _kv()
    lens = [1, R - 1, R, R + 1, 2 * R + 63]
    case = Case(kv, len(lens), 3, 3 * R, lens, seed=R)
    q = case.queries(len(lens))
    cache, table = case.paged(R, dev)
    cur = _dev(np.array(lens, dtype=np.int32) - 1, dev)
    for S in (0, 3, -64):
        out = torch.empty(len(lens), 3, HS, dtype=torch.bfloat16, device=dev)
        ws = kvattn.Workspace(len(lens), 3, 3 * R, S)
        kvattn.paged_decode(out, _qkv(q, dev), cache, len(lens), 3, HS, kv_dtype=kv, cur_len=cur, lens_per_seq=True, S=S,
                            **ws.kwargs())
        case.check(out.float().cpu().numpy(), q, [(b, b, T) for b, T in enumerate(lens)], f"R {R} S {S}")


@pytest.mark.parametrize("kv", KV4)
@pytest.mark.parametrize("B,NH,n", [(260, 4, 96), (260, 4, 95), (129, 2, 96), (128, 2, 128), (300, 1, 200)])
def test_workspace_of_ragged_batches(dev, kv, B, NH, n):
    """The plan is that of one length for the batch: its workspace serves such a batch.  Per-sequence lengths of many
    heads may need more; the workspace for every choice (S = 0) serves them too."""
    import torch
    kvattn = _kv()
    R = 64
    case = Case(kv, 3, NH, n * R, [n * R, 1, 300], seed=18)
    few, table = case.paged(R, dev)
    own = np.arange(B) % 3
    cache = kvattn.PagedCache(few.pages, _dev(table[own], dev), n, R, few.num_pages, few.page_scales)
    q = case.queries(B)
    lens = np.array(case.lens, np.int32)[own]
    planned = kvattn.plan(B, NH, HS, n * R, kv_dtype=kv)[1]
    tokens = [(b, b % 3, int(lens[b])) for b in range(0, B, 7)]

    def call(S, cur, per_seq):
        out = torch.full((B, NH, HS), 7.0, dtype=torch.bfloat16, device=dev)
        ws = kvattn.Workspace(B, NH, n * R, S)
        kvattn.paged_decode(out, _qkv(q, dev), cache, B, NH, HS, kv_dtype=kv, cur_len=cur, lens_per_seq=per_seq, **ws.kwargs())
        return out.float().cpu().numpy()
    case.check(call(0, _dev(lens - 1, dev), True), q, tokens, "ragged")
    case.check(call(planned, _dev(np.array([299], np.int32), dev), False), q, [(b, b % 3, 300) for b in range(0, B, 21)], "one")
    if B * NH > 256 and n >= 96 and n // 32 > planned:
        with pytest.raises(kvattn.KvAttnError) as e:
            call(planned, _dev(lens - 1, dev), True)
        assert e.value.status == kvattn.ERR_WORKSPACE
    else:
        case.check(call(planned, _dev(lens - 1, dev), True), q, tokens, "ragged, as planned")


@pytest.mark.parametrize("kv", KV4)
def test_bad_pages_are_skipped(dev, kv):
    """Positions of table entries outside the pool do not count; a sequence with none left gives zero."""
    import torch
    kvattn = _kv()
    case = Case(kv, 3, 2, 192, [192, 130, 64], seed=12)
    q = case.queries(3)
    cache, table = case.paged(64, dev)
    cache.block_table[0, 1] = -1
    cache.block_table[1, 0] = cache.num_pages
    cache.block_table[2, 0] = 2 ** 31 - 1
    out = torch.empty(3, 2, HS, dtype=torch.bfloat16, device=dev)
    ws = kvattn.Workspace(3, 2, 192)
    kvattn.paged_decode(out, _qkv(q, dev), cache, 3, 2, HS, kv_dtype=kv, lens_per_seq=True,
                        cur_len=torch.tensor([191, 129, 63], dtype=torch.int32, device=dev), **ws.kwargs())
    got = out.float().cpu().numpy()
    keep = {0: np.r_[0:64, 128:192], 1: np.r_[64:130], 2: np.r_[0:0]}
    for b, rows in keep.items():
        for h in range(2):
            k, v = (kv4ref.decode(case.packed[i, b, h, rows], case.scale[i, b, h, rows], kv) for i in (0, 1))
            ref, wv = kv4ref.attend(q[b, h].astype(np.float64), k, v, len(rows))
            lim = kv4ref.bound(ref, wv, q[b, h], case.scale[0, b, h, rows], case.scale[1, b, h, rows], kv, len(rows))
            assert (np.abs(got[b, h] - ref) <= lim).all(), (b, h)


@pytest.mark.parametrize("kv", KV4)
@pytest.mark.parametrize("counts", [[1], [8], [9], [17], [3, 0, 1, 8, 0, 12, 2]])
@pytest.mark.parametrize("S", [0, 5])
def test_paged_decode_tokens(dev, kv, counts, S):
    """Several tokens a sequence (none, groups of eight and more), rows behind the last as they were."""
    import torch
    kvattn = _kv()
    R, n = 64, 6
    r = np.random.RandomState(len(counts))
    lens = [int(r.randint(max(c, 1), n * R + 1)) for c in counts]
    lens[0] = n * R
    case = Case(kv, len(counts), 2, n * R, lens, seed=13)
    N, spare = sum(counts), 3
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = case.queries(N + spare)
    cache, _ = case.paged(R, dev)
    out = torch.full((N + spare, 2, HS), 7.0, dtype=torch.bfloat16, device=dev)
    ws = kvattn.Workspace(N + spare, 2, n * R, S)
    kvattn.paged_decode_tokens(out, _qkv(q, dev), cache, _dev(start, dev), _dev(np.array(lens, np.int32), dev), len(counts),
                               N + spare, 2, HS, kv_dtype=kv, max_new=max(counts), S=S, **ws.kwargs())
    got = out.float().cpu().numpy()
    tokens = [(start[b] + i, b, lens[b] - c + i + 1) for b, c in enumerate(counts) for i in range(c)]
    case.check(got, q, tokens, f"counts {counts}")
    assert (got[N:] == 7.0).all()


@pytest.mark.parametrize("kv", KV4)
@pytest.mark.parametrize("counts", [[1, 1, 1], [2, 4, 0], [3, 8, 1], [1] * 140, [3, 0, 1, 2] * 35, [5, 1] * 70,
                                    [5, 0, 1] * 90])
def test_paged_decode_tokens_large_pool(dev, kv, counts):
    """A pool of more than 128 MiB, of which the loads are others (as read only once), and room for 320000
    positions a sequence; no bound on the tokens of one."""
    import torch
    kvattn = _kv()
    R, NH, P, room = 64, 2, 15000, 5000
    B, N = len(counts), sum(counts)
    case = Case(kv, B, NH, 256, ([256, 65, 130] + [9 + i for i in range(B)])[:B], seed=16)
    q = case.queries(N)
    small, table = case.paged(R, dev)
    front = P - small.num_pages             # the rows lie in the last pages
    pages = torch.full((P, 2, NH, R, HS // 2), 0xFF, dtype=torch.uint8, device=dev)
    scales = torch.full((P, 2, NH, R), float("nan"), dtype=torch.float32, device=dev)
    pages[front:], scales[front:] = small.pages, small.page_scales
    wide = np.full((B, room), -1, dtype=np.int32)
    wide[:, :table.shape[1]] = table + front
    cache = kvattn.PagedCache(pages, _dev(wide, dev), room, R, P, scales)
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    tokens = [(start[b] + i, b, case.lens[b] - c + i + 1) for b, c in enumerate(counts) for i in range(c)]
    ws = kvattn.Workspace(N, NH, room * R)
    for most in (max(counts), 2 ** 31 - 1):
        out = torch.full((N, NH, HS), 7.0, dtype=torch.bfloat16, device=dev)
        kvattn.paged_decode_tokens(out, _qkv(q, dev), cache, _dev(start, dev), _dev(np.array(case.lens, np.int32), dev), B, N,
                                   NH, HS, kv_dtype=kv, max_new=most, **ws.kwargs())
        case.check(out.float().cpu().numpy(), q, tokens, f"counts {counts} most {most}")


@pytest.mark.parametrize("kv", KV4)
@pytest.mark.parametrize("B,counts,lead", [(3, [1, 0, 2], 20), (64, [3, 0, 9, 1], 0), (65, [8], 5), (300, [0, 0, 0, 17], 9),
                                           (4096, [4, 0, 8, 1, 7], 0), (4097, [1, 0, 0], 8), (5000, [3, 2, 4], 100),
                                           (1024, [8], 0)])
@pytest.mark.parametrize("S", [0, 2])
def test_paged_decode_tokens_of_any_number(dev, kv, B, counts, lead, S):
    """max_new that says nothing, over batches of every size: sequences share their first pages, as prompts may, and
    the tokens may begin behind rows of another use, which are left as they were."""
    import torch
    kvattn = _kv()
    R, n, own = 64, 2, 16
    case = Case(kv, own, 2, n * R, [128, 70, 64, 9] * 4, seed=17)
    counts = (counts * B)[:B]
    counts[B // 2] = 23                             # one with three groups
    start = lead + np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    N, spare = int(start[-1]), 3
    q = case.queries(N + spare)
    few, table = case.paged(R, dev)
    cache = kvattn.PagedCache(few.pages, _dev(table[np.arange(B) % own], dev), n, R, few.num_pages, few.page_scales)
    lens = np.array(case.lens, np.int32)[np.arange(B) % own]
    ws = kvattn.Workspace(N + spare, 2, n * R)
    tokens = [(start[b] + i, b % own, lens[b] - c + i + 1) for b, c in enumerate(counts) for i in range(c)]
    for most in (23, 2 ** 31 - 1):
        out = torch.full((N + spare, 2, HS), 7.0, dtype=torch.bfloat16, device=dev)
        kvattn.paged_decode_tokens(out, _qkv(q, dev), cache, _dev(start, dev), _dev(lens, dev), B, N + spare, 2, HS, kv_dtype=kv,
                                   max_new=most, S=S, **ws.kwargs())
        got = out.float().cpu().numpy()
        assert (got[:lead] == 7.0).all() and (got[N:] == 7.0).all() and not (got[lead:N] == 7.0).all(-1).any()
        case.check(got, q, tokens[::1 + len(tokens) // 1500], f"B {B} most {most}")
        case.check(got, q, [t for t in tokens if t[0] >= start[B // 2] and t[0] < start[B // 2 + 1]], f"B {B} most {most}")


@pytest.mark.parametrize("kv", KV4)
def test_tokens_see_nothing_of_later_ones(dev, kv):
    """A later draft's row of infinite or NaN scale leaves the tokens before it as they are; tokens
    before the first position attend nothing and give zero."""
    import torch
    kvattn = _kv()
    case = Case(kv, 2, 1, 128, [100, 2], seed=14)
    q = case.queries(8)
    case.scale[0, 0, 0, 98], case.scale[1, 0, 0, 98] = np.nan, np.inf      # row of token 2 of sequence 0
    cache, _ = case.paged(64, dev)
    out = torch.full((8, 1, HS), 7.0, dtype=torch.bfloat16, device=dev)
    ws = kvattn.Workspace(8, 1, 128)
    # Sequence 0: 4 tokens behind 96 positions; sequence 1: 4 tokens, but only 2 positions.
    kvattn.paged_decode_tokens(out, _qkv(q, dev), cache, _dev(np.array([0, 4, 8], np.int32), dev),
                               _dev(np.array([100, 2], np.int32), dev), 2, 8, 1, HS, kv_dtype=kv, max_new=4, **ws.kwargs())
    got = out.float().cpu().numpy()
    clean = Case(kv, 2, 1, 128, [100, 2], seed=14)
    clean.check(got, q, [(0, 0, 97), (1, 0, 98), (4, 1, -1), (5, 1, 0), (6, 1, 1), (7, 1, 2)], "masked rows")
    assert np.isnan(got[2]).any() and np.isnan(got[3]).any()
    assert (got[4:6] == 0).all()


@pytest.mark.parametrize("kv", KV4)
def test_tokens_wrong_starts_stay_inside(dev, kv):
    """Offsets beyond the tokens are clamped: no row behind num_tokens is read or written."""
    import torch
    kvattn = _kv()
    case = Case(kv, 2, 1, 64, [64, 64], seed=15)
    q = case.queries(4)
    cache, _ = case.paged(64, dev)
    out = torch.full((6, 1, HS), 7.0, dtype=torch.bfloat16, device=dev)
    ws = kvattn.Workspace(4, 1, 64)
    kvattn.paged_decode_tokens(out, _qkv(q, dev), cache, _dev(np.array([-3, 2, 90], np.int32), dev),
                               _dev(np.array([64, 1000], np.int32), dev), 2, 4, 1, HS, kv_dtype=kv, max_new=8, **ws.kwargs())
    got = out.float().cpu().numpy()
    case.check(got, q, [(0, 0, 63), (1, 0, 64), (2, 1, 63), (3, 1, 64)], "clamped starts")
    assert (got[4:] == 7.0).all()


# ------------------------------------------------------------------------------------
# The append.
# ------------------------------------------------------------------------------------
def _append_rows(seed):
    """bf16 rows: normal ones, ties on code boundaries, zeros, the smallest and largest values,
    infinities and NaN."""
    r = np.random.RandomState(seed)
    rows = [r.standard_normal(HS) * 10.0 ** r.randint(-6, 6) for _ in range(8)]
    for top in (7.0, 6.0, 1.75, 96.0):
        x = r.choice([0.0, 0.125, 0.25, 0.5, 0.75, -0.5, -0.125, 1 / 3, 1.0], HS) * top
        x[r.randint(HS)] = top
        rows.append(x)
    rows += [np.zeros(HS), -np.zeros(HS), 1e-39 * r.standard_normal(HS), 3e38 * np.sign(r.standard_normal(HS))]
    for special in (np.inf, -np.inf, np.nan):
        x = r.standard_normal(HS)
        x[r.randint(HS)] = special
        rows.append(x)
    return _bf16(np.stack(rows))


@pytest.mark.parametrize("kv", KV4)
@pytest.mark.parametrize("paged", [False, True])
def test_append_codes(dev, kv, paged):
    """Codes and scales of the append, bit for bit; nothing else of the cache changes."""
    import torch
    kvattn = _kv()
    rows = _append_rows(1)
    B, NH, maxT = rows.shape[0], 2, 128
    qkv = torch.full((B, 3, NH, HS), 0.5, dtype=torch.bfloat16, device=dev)
    src = np.stack([np.stack([rows, np.roll(rows, 1, 0)], 1), np.stack([np.roll(rows, 2, 0), np.roll(rows, 3, 0)], 1)], 1)
    qkv[:, 1:] = _dev(src, dev, torch.bfloat16)                            # [B, 2, NH, 64]
    lens = np.array([(11 * i) % maxT for i in range(B)], dtype=np.int32)
    want_c, want_s = kv4ref.encode(src, kv)
    if paged:
        table = np.random.RandomState(2).permutation(2 * B).reshape(B, 2).astype(np.int32)
        shape = (2 * B, 2, NH, 64)
        at = [(table[b, lens[b] // 64], slice(None), slice(None), lens[b] % 64) for b in range(B)]
    else:
        shape = (2, B, NH, maxT)
        at = [(slice(None), b, slice(None), lens[b]) for b in range(B)]
    codes = torch.full(shape + (HS // 2,), 0x5A, dtype=torch.uint8, device=dev)
    scale = torch.full(shape, -3.0, device=dev)
    cur = _dev(lens, dev)
    if paged:
        cache = kvattn.PagedCache(codes, _dev(table, dev), 2, 64, 2 * B, scale)
        kvattn.paged_cache_write(cache, qkv, B, NH, HS, kv_dtype=kv, cur_len=cur, lens_per_seq=True)
    else:
        kvattn.kv_cache_write(codes, qkv, B, NH, HS, maxT, kv_dtype=kv, kv_scale=scale, cur_len=cur, lens_per_seq=True)
    got_c, got_s = codes.cpu().numpy(), scale.cpu().numpy()
    exp_c, exp_s = np.full_like(got_c, 0x5A), np.full_like(got_s, -3.0)
    for b in range(B):
        exp_c[at[b]], exp_s[at[b]] = want_c[b], want_s[b]
    assert np.array_equal(got_s.view(np.uint32), exp_s.view(np.uint32))
    assert np.array_equal(got_c, exp_c)


@pytest.mark.parametrize("kv", KV4)
@pytest.mark.parametrize("paged", [False, True])
def test_append_decode_equals_two_calls(dev, kv, paged):
    import torch
    kvattn = _kv()
    lens = [1, 64, 129, 192]
    case = Case(kv, 4, 3, 192, lens, seed=21)
    qkv = _dev(_bf16(case.r.standard_normal((4, 3, 3, HS))), dev, torch.bfloat16)
    cur = _dev(np.array(lens, np.int32) - 1, dev)
    ws = kvattn.Workspace(4, 3, 192)
    outs, caches = [], []
    for fused in (False, True):
        out = torch.empty(4, 3, HS, dtype=torch.bfloat16, device=dev)
        if paged:
            cache, _ = case.paged(64, dev)
            c, s = cache.pages, cache.page_scales
            if not fused:
                kvattn.paged_cache_write(cache, qkv, 4, 3, HS, kv_dtype=kv, cur_len=cur, lens_per_seq=True)
            kvattn.paged_decode(out, qkv, cache, 4, 3, HS, kv_dtype=kv, cur_len=cur, lens_per_seq=True, append=fused,
                                **ws.kwargs())
        else:
            c, s = _dev(case.packed, dev), _dev(case.scale, dev)
            kw = dict(kv_dtype=kv, kv_scale=s, cur_len=cur, lens_per_seq=True)
            if not fused:
                kvattn.kv_cache_write(c, qkv, 4, 3, HS, 192, **kw)
            (kvattn.append_decode if fused else kvattn.decode)(out, qkv, c, 4, 3, HS, 192, **kw, **ws.kwargs())
        outs.append(out)
        caches.append((c, s))
    assert torch.equal(outs[0], outs[1]) and not torch.isnan(outs[0].float()).any()
    assert torch.equal(caches[0][0], caches[1][0])
    assert torch.equal(caches[0][1].view(torch.int32), caches[1][1].view(torch.int32))


def test_refused_append_decode_appends_nothing(dev):
    import torch
    kvattn = _kv()
    codes = torch.zeros(2, 1, 2, 4096, HS // 2, dtype=torch.uint8, device=dev)
    scale = torch.zeros(2, 1, 2, 4096, device=dev)
    qkv = torch.ones(1, 3, 2, HS, dtype=torch.bfloat16, device=dev)
    out = torch.empty(1, 2, HS, dtype=torch.bfloat16, device=dev)
    cur = torch.zeros(1, dtype=torch.int32, device=dev)
    with pytest.raises(kvattn.KvAttnError):
        kvattn.append_decode(out, qkv, codes, 1, 2, HS, 4096, kv_dtype="int4", kv_scale=scale, cur_len=cur, S=8)
    assert not codes.any() and not scale.any()


# ------------------------------------------------------------------------------------
# How calls are made.
# ------------------------------------------------------------------------------------
@pytest.mark.parametrize("kv", KV4)
def test_repeats_are_bit_identical_on_a_used_workspace(dev, kv):
    """The order in which segments finish does not change a result, and other plans on the same workspace
    in between leave its counters at zero."""
    import torch
    kvattn = _kv()
    case = Case(kv, 2, 4, 2048, [2048, 1500], seed=30)
    q = case.queries(2)
    ws = kvattn.Workspace(2, 4, 2048)
    codes, scale, qkv = _dev(case.packed, dev), _dev(case.scale, dev), _qkv(q, dev)
    cur = _dev(np.array([2047, 1499], np.int32), dev)
    first = None
    for i in range(30):
        out = torch.empty(2, 4, HS, dtype=torch.bfloat16, device=dev)
        for S in (3, 0, 16):
            o = torch.empty(2, 4, HS, dtype=torch.bfloat16, device=dev)
            kvattn.decode(o, qkv, codes, 2, 4, HS, 2048, kv_dtype=kv, kv_scale=scale, cur_len=cur, lens_per_seq=True, S=S,
                          **ws.kwargs())
            out = o if S == 16 else out
        first = out if first is None else first
        assert torch.equal(out, first)
    case.check(first.float().cpu().numpy(), q, [(0, 0, 2048), (1, 1, 1500)], "repeats")


@pytest.mark.parametrize("kv", KV4)
def test_captured_step(dev, kv):
    """Append and attention captured once, replayed while the length grows on the device, with eager work
    between the replays: every replay equals the eager calls."""
    import torch
    kvattn = _kv()
    case = Case(kv, 2, 2, 256, [256, 256], seed=31)
    qkv = torch.empty(2, 3, 2, HS, dtype=torch.bfloat16, device=dev)
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    out = torch.empty(2, 2, HS, dtype=torch.bfloat16, device=dev)
    caches = [(_dev(case.packed, dev), _dev(case.scale, dev)) for _ in range(2)]
    ws = [kvattn.Workspace(2, 2, 256, 4) for _ in range(2)]

    def step(i, o):
        c, s = caches[i]
        kvattn.append_decode(o, qkv, c, 2, 2, HS, 256, kv_dtype=kv, kv_scale=s, cur_len=lens, lens_per_seq=True, S=4,
                             **ws[i].kwargs())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(0, out)
    for t in range(6):
        qkv.copy_(torch.randn(2, 3, 2, HS, generator=torch.Generator().manual_seed(t)))
        lens.copy_(torch.tensor([40 * t, 51 * t]))
        eager = torch.empty_like(out)
        step(1, eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert torch.equal(caches[0][0], caches[1][0])


@pytest.mark.parametrize("kv", KV4)
def test_rows_past_32_bit_offsets(dev, kv):
    """Pages whose bytes lie beyond 4 GiB of the pool, and beyond 2^31 rows' worth of elements."""
    import torch
    kvattn = _kv()
    R, NH = 4096, 12
    page = 2 * NH * R * HS // 2
    P = (5 << 30) // page
    case = Case(kv, 1, NH, R, [200], seed=33)
    q = case.queries(1)
    pages = torch.empty(P, 2, NH, R, HS // 2, dtype=torch.uint8, device=dev)
    scales = torch.empty(P, 2, NH, R, device=dev)
    pages[P - 1] = _dev(case.packed[:, 0], dev)
    scales[P - 1] = _dev(case.scale[:, 0], dev)
    cache = kvattn.PagedCache(pages, torch.tensor([[P - 1]], dtype=torch.int32, device=dev), 1, R, P, scales)
    out = torch.empty(1, NH, HS, dtype=torch.bfloat16, device=dev)
    ws = kvattn.Workspace(1, NH, R)
    kvattn.paged_decode(out, _qkv(q, dev), cache, 1, NH, HS, kv_dtype=kv,
                        cur_len=torch.tensor([199], dtype=torch.int32, device=dev), **ws.kwargs())
    case.check(out.float().cpu().numpy(), q, [(0, 0, 200)], "far page")
    # Store and load there.
    slots = torch.arange(3, dtype=torch.int64, device=dev) + (P - 1) * R + 1000
    qkv = torch.randn(3, 3, NH, HS, device=dev).to(torch.bfloat16)
    back = torch.empty(3, 2, NH, HS, dtype=torch.bfloat16, device=dev)
    kvattn.paged_store(cache, qkv, slots, 3, NH, HS, kv_dtype=kv)
    kvattn.paged_load(back, cache, slots, 3, NH, HS, kv_dtype=kv)
    c, s = kv4ref.encode(qkv[:, 1:].float().cpu().numpy(), kv)
    assert torch.equal(pages[P - 1, :, :, 1000:1003].permute(2, 0, 1, 3).cpu(), torch.from_numpy(c))
    want = (kv4ref.decode(c, np.ones_like(s), kv).astype(np.float32) * s[..., None])
    assert torch.equal(back.cpu(), torch.from_numpy(want).to(torch.bfloat16))


@pytest.mark.parametrize("T,n", [(1, 1), (64, 1), (999, 1), (999, 5), (2048, 8), (4097, 1)])
def test_int4_within_its_operands_bound(dev, monkeypatch, T, n):
    """The INT4 operand is code + 8, of magnitude 1 to 15: the bound of sums over such terms, half as wide as one for
    another operand's 31."""
    import torch
    kvattn = _kv()
    monkeypatch.setitem(kv4ref.BIAS, "int4", 8.0)
    maxT = -(-T // 64) * 64
    case = Case("int4", 2, 3, maxT, [T, max(n, T // 2)], seed=T + n, sharp=2.0)
    cache, _ = case.paged(64, dev)
    q = case.queries(2 * n)
    out = torch.empty(2 * n, 3, HS, dtype=torch.bfloat16, device=dev)
    ws = kvattn.Workspace(2 * n, 3, maxT)
    kvattn.paged_decode_tokens(out, _qkv(q, dev), cache, _dev(np.array([0, n, 2 * n], np.int32), dev),
                               _dev(np.array(case.lens, np.int32), dev), 2, 2 * n, 3, HS, kv_dtype="int4", max_new=n, **ws.kwargs())
    tokens = [(b * n + i, b, case.lens[b] - n + i + 1) for b in range(2) for i in range(n)]
    case.check(out.float().cpu().numpy(), q, tokens, f"T {T} n {n}")
