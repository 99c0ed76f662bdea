"""Penalties, biases and grammar masks on logits, and their probabilities, against a row-by-row restatement in 64 bits
(treeref.rules, treeref.softmax)."""
import numpy as np
import pytest

import treeref

pytestmark = pytest.mark.gpu


def _kv():
    from cuda_gpt2_inference_amd import kvattn
    return kvattn


def _dev(x, dev):
    import torch
    x = np.ascontiguousarray(x)
    return torch.from_numpy(x.view(np.int64) if x.dtype == np.uint64 else x).to(dev)


class Case:
    def __init__(self, seed, sizes, V, stride, dtype, history=0, bias=0, grammar=False, branches=False, penalties=True,
                 temperature=True, wide_ids=False):
        r = np.random.RandomState(seed)
        self.r, self.V, self.stride, self.dtype, self.B = r, V, stride, dtype, len(sizes)
        self.start, self.parents = treeref.forest(r, sizes)
        self.N = N = len(self.parents)
        self.x = np.full((N, stride), np.nan, dtype=np.float32)        # what lies behind the vocabulary is not read
        self.x[:, :V] = 3.0 * r.standard_normal((N, V))
        if dtype == "bf16":
            self.x = treeref.bf16(self.x)
        B = self.B
        ids = lambda *s: (r.randint(-3, V + 3, s) if wide_ids else (V * r.rand(*s) ** 3).astype(int)).astype(np.int32)   # noqa: E731
        f = lambda x: x.astype(np.float32)                              # noqa: E731
        self.rules = {}
        self.history = ids(B, history) if history else None
        if history:
            self.rules.update(history=self.history, history_len=r.randint(0, history + 1, B).astype(np.int32), max_history=history,
                              prompt_len=r.randint(0, history + 1, B).astype(np.int32))
        if penalties:
            self.rules.update(repetition=f(1 + 0.5 * r.rand(B)), frequency=f(r.rand(B) - 0.3), presence=f(r.rand(B) - 0.3))
        if branches:
            masks, _ = treeref.masks(self.start, self.parents, 2)
            self.rules.update(tokens=ids(N), masks=masks, mask_words=2)
        if bias:
            n = r.randint(0, bias + 1, B)
            self.rules.update(bias_start=np.concatenate([[0], np.cumsum(n)]).astype(np.int32), bias_ids=ids(n.sum()),
                              bias=f(4 * r.standard_normal(n.sum())), num_bias=int(n.sum()), max_bias=bias)
        if grammar:
            words = (V + 31) // 32 + 1
            self.rules.update(allowed=r.randint(0, 1 << 32, (3, words), dtype=np.uint32).view(np.int32), num_allowed=3,
                              allowed_stride=words, allowed_of=r.randint(-1, 4, N).astype(np.int32))
        if temperature:
            self.rules["temperature"] = f(np.where(r.rand(B) < 0.25, 0.0, 0.3 + r.rand(B)))

    def row(self, t):
        """The row's rules in 64 bits."""
        g = self.rules
        b = int(np.searchsorted(self.start[1:], t, side="right"))
        held, made, bias, allowed = [], [], {}, None
        if "history" in g:
            n = int(g["history_len"][b])
            h = g["history"][b, :n].tolist()
            held, made = list(h), h[int(g["prompt_len"][b]):] if "prompt_len" in g else list(h)
        if "masks" in g:
            own = [int(g["tokens"][self.start[b] + j]) for j in range(128)
                   if (int(g["masks"][t, j >> 6]) >> (j & 63)) & 1]
            held, made = held + own, made + own
        if "bias" in g:
            for e in range(int(g["bias_start"][b]), int(min(g["bias_start"][b + 1], g["bias_start"][b] + g["max_bias"]))):
                bias[int(g["bias_ids"][e])] = float(g["bias"][e])
        if "allowed" in g and 0 <= (g["allowed_of"][t] if "allowed_of" in g else t) < g["num_allowed"]:
            line = g["allowed"][g["allowed_of"][t] if "allowed_of" in g else t].view(np.uint32)
            v = np.arange(self.V)
            allowed = ((line[v // 32] >> (v % 32).astype(np.uint32)) & 1).astype(bool)
        one = lambda k, d: float(g[k][b]) if k in g else d             # noqa: E731
        x, err = treeref.rules(self.x[t, :self.V], held, made, one("repetition", 1.0), one("frequency", 0.0), one("presence", 0.0),
                               bias, allowed)
        return x, err, one("temperature", 1.0)

    def run(self, dev, out_dtype, probs, spare=2, out_stride=None, offset=0):
        import torch
        kvattn = _kv()
        td = {"f32": torch.float32, "bf16": torch.bfloat16}
        rows, so = self.N + spare, out_stride or self.stride
        flat = torch.zeros(rows * self.stride + offset, dtype=td[self.dtype], device=dev)
        x = flat[offset:].view(rows, self.stride)
        x[:self.N] = torch.from_numpy(self.x).to(td[self.dtype]).to(dev)
        out = torch.full((rows, so), 55.0, dtype=td[out_dtype], device=dev)
        dev_rules = {k: _dev(v, dev) if isinstance(v, np.ndarray) else v for k, v in self.rules.items()}
        if not probs:
            dev_rules.pop("temperature", None)
        # (Arrays of a line a row have lines for the spare rows too.)
        for k in ("tokens", "masks", "allowed_of"):
            if k in dev_rules:
                dev_rules[k] = torch.cat([dev_rules[k], torch.zeros_like(dev_rules[k][:spare])])
        kvattn.process_logits(out, x, kvattn.LogitRules(**dev_rules) if dev_rules else None, _dev(self.start, dev), self.B, rows,
                              self.V, row_stride=self.stride, out_stride=so, dtype=self.dtype, out_dtype=out_dtype, probs=probs)
        assert (out[self.N:] == 55.0).all() and (out[:, self.V:] == 55.0).all()
        return out[:self.N, :self.V].double().cpu().numpy()

    def check(self, dev, out_dtype="f32", probs=True, **kw):
        got = self.run(dev, out_dtype, probs, **kw)
        half = treeref.HALF_STEP[out_dtype]
        for t in range(self.N):
            x, err, T = self.row(t)
            if probs:
                x, err = treeref.softmax(x, err, T)
            with np.errstate(invalid="ignore"):
                ok = (np.abs(got[t] - x) <= err + half * np.abs(x) + 2.0 ** -126) | (got[t] == x)
            assert ok.all(), (t, np.nonzero(~ok)[0][:5], got[t][~ok][:5], x[~ok][:5])
            if probs and T > 0 and x.any() and out_dtype == "f32":
                assert abs(got[t].sum() - 1) < 1e-5


VOCABULARIES = [(1, 1), (5, 7), (31, 32), (33, 36), (1000, 1001), (50257, 50304), (60000, 60000)]


@pytest.mark.parametrize("V,stride", VOCABULARIES)
@pytest.mark.parametrize("dtype,out_dtype,probs", [("f32", "f32", True), ("bf16", "f32", True), ("f32", "bf16", False),
                                                   ("bf16", "bf16", True), ("f32", "f32", False)])
def test_all_rules(dev, V, stride, dtype, out_dtype, probs):
    c = Case(V + len(dtype), [3, 0, 1, 70] if V < 2000 else [2, 0, 3], V, stride, dtype, history=200, bias=12, grammar=True,
             branches=True)
    c.check(dev, out_dtype, probs)


@pytest.mark.parametrize("kw", [dict(), dict(history=1), dict(history=5000), dict(bias=400), dict(grammar=True), dict(branches=True),
                                dict(history=50, penalties=False), dict(history=700, bias=30, wide_ids=True, branches=True),
                                dict(temperature=False, grammar=True)])
@pytest.mark.parametrize("probs", [True, False])
def test_each_rule(dev, kw, probs):
    Case(7, [4, 1, 2], 3001, 3001, "f32", **kw).check(dev, "f32", probs)


def test_no_prompt_and_no_lines(dev):
    """Without prompt_len all of the history was generated; without allowed_of a row has its own line."""
    c = Case(8, [1, 1, 1], 500, 500, "f32", history=90, grammar=True)
    del c.rules["prompt_len"]
    c.rules["allowed_of"] = np.arange(3, dtype=np.int32)
    want = c.run(dev, "f32", True, spare=0)
    c.check(dev)
    del c.rules["allowed_of"]
    assert np.array_equal(c.run(dev, "f32", True, spare=0), want)


@pytest.mark.parametrize("offset,out_stride", [(0, 1003), (1, 1004), (3, 1001)])
def test_unaligned(dev, offset, out_stride):
    for dtype in ("f32", "bf16"):
        Case(9, [2, 3], 1001, 1004, dtype, history=30, grammar=True).check(dev, "bf16", True, offset=offset, out_stride=out_stride)


def test_many_sequences(dev):
    """Rows find their sequence among many, of which some have none."""
    sizes = [(i * 7) % 3 for i in range(5000)]
    c = Case(10, sizes, 40, 40, "f32", history=6, bias=2, branches=True)
    c.check(dev)


def test_rows_without_starts(dev):
    import torch
    kvattn = _kv()
    c = Case(11, [1] * 6, 700, 700, "f32", history=40)
    want = c.run(dev, "f32", True, spare=0)
    x = torch.from_numpy(c.x).to(dev)
    rules = kvattn.LogitRules(**{k: _dev(v, dev) if isinstance(v, np.ndarray) else v for k, v in c.rules.items()})
    kvattn.process_logits(x, x, rules, None, 6, 6, 700)                  # in place
    assert np.array_equal(x.double().cpu().numpy(), want)


@pytest.mark.parametrize("V", [900, 60000])
def test_strange_logits(dev, V):
    """Everything forbidden; NaN and infinities at forbidden tokens; ties; equal logits; -inf; allowed NaN and inf."""
    import torch
    kvattn = _kv()
    x = torch.randn(8, V, device=dev)
    allowed = torch.full((8, (V + 31) // 32), -1, dtype=torch.int32, device=dev)
    allowed[0] = 0
    x[1, 32:64] = torch.tensor([float("nan"), float("inf")], device=dev).repeat(16)
    allowed[1, 1] = 0
    x[2, 5] = x[2, 700] = 50.0
    x[3] = -3.0
    x[4] = float("-inf")
    x[5, 9:] = float("-inf")
    x[6, 17] = float("nan")
    x[7, 18] = float("inf")
    for T in (0.0, 0.7):
        t = torch.full((8,), T, device=dev)
        rules = kvattn.LogitRules(allowed=allowed, num_allowed=8, allowed_stride=allowed.shape[1], temperature=t)
        out = torch.full((8, V), 9.0, device=dev)
        kvattn.process_logits(out, x, rules, None, 8, 8, V)
        assert (out[0] == 0).all() and (out[4] == 0).all()
        clean = x[1].clone()
        clean[32:64] = float("-inf")
        if T:
            assert torch.allclose(out[1], torch.softmax(clean.double() / float(t[0]), 0).float(), rtol=1e-5, atol=0)
            assert out[2].argmax() in (5, 700) and out[2, 5] == out[2, 700] and torch.isfinite(out[2]).all()
            # Equal weights: their sum is exact up to 2^24, a quotient and a product round.
            assert ((out[3].double() * V - 1).abs() <= 2 * 2.0 ** -24).all()
            assert (out[5, 9:] == 0).all() and abs(float(out[5].sum()) - 1) < 1e-6
            assert torch.isnan(out[6]).any() and torch.isnan(out[7]).any()
        else:
            assert out[1].argmax() == clean.argmax() and out[1].sum() == 1
            assert out[2, 5] == 1 and out[2].sum() == 1 and out[3, 0] == 1 and out[3].sum() == 1
            assert out[7, 18] == 1 and out[7].sum() == 1


def test_temperature_extremes(dev):
    import torch
    kvattn = _kv()
    x = torch.randn(3, 2000, device=dev) * 10
    rules = kvattn.LogitRules(temperature=torch.tensor([1e-4, 1e4, float("nan")], device=dev))
    out = torch.empty_like(x)
    kvattn.process_logits(out, x, rules, None, 3, 3, 2000)
    want = torch.softmax(x.double() / torch.tensor([[1e-4], [1e4], [1.0]], device=dev, dtype=torch.float64), -1)
    # An exponent of 80 / T in base 2 rounds four times; of the first row only the first tokens weigh anything.
    assert ((out[1].double() - want[1]).abs() <= 1e-5 * want[1]).all()
    assert float((out[0].double() - want[0]).abs().max()) < 1e-2 and out[0].argmax() == x[0].argmax()
    assert out[2].sum() == 1 and out[2].argmax() == x[2].argmax()


def _same(c, dev, probs=True, dtype="f32", **extra):
    """A call's output as bits."""
    import torch
    kvattn = _kv()
    x = torch.zeros((c.N, c.stride), device=dev)
    x[:] = torch.from_numpy(np.nan_to_num(c.x)).to(dev)
    out = torch.zeros((c.N, c.stride), device=dev)
    rules = {k: _dev(v, dev) if isinstance(v, np.ndarray) else v for k, v in c.rules.items()}
    rules.update(extra)
    kvattn.process_logits(out, x, kvattn.LogitRules(**rules), _dev(c.start, dev), c.B, c.N, c.V, row_stride=c.stride, out_stride=c.stride,
                          probs=probs)
    return out.cpu()


@pytest.mark.parametrize("V", [3001, 50257])
def test_slices_that_wait_in_vain(dev, V):
    """Every slice works the others out itself: the same bits."""
    import torch
    kvattn = _kv()
    c = Case(20, [2, 1, 3], V, V + 3, "f32", history=300, bias=9, grammar=True, branches=True)
    want = _same(c, dev)
    before = kvattn.set_merge_poll_limit(0)
    try:
        got = _same(c, dev)
        torch.cuda.synchronize()
    finally:
        kvattn.set_merge_poll_limit(before)
    assert torch.equal(got, want)


def test_without_a_workspace(dev):
    """A row by one workgroup: the same mathematics in another order."""
    c = Case(21, [3, 2], 50257, 50304, "f32", history=300, grammar=True, branches=True)
    c.check(dev)
    c.rules["workspace"] = None
    c.check(dev)
    c.check(dev, "bf16")


@pytest.mark.parametrize("rows", [100, 200, 300, 700])
def test_many_rows(dev, rows):
    """Every number of slices, and a row a workgroup."""
    c = Case(22, [rows // 2, 0, rows - rows // 2], 9001, 9004, "f32", history=20, bias=3)
    c.check(dev)
    c = Case(22, [rows], 33000, 33000, "bf16", history=20)
    c.check(dev, "bf16", probs=rows != 200)


def test_histories_that_do_not_fit_one_workgroup(dev):
    """Rows at a time; refused where slices cannot be."""
    import torch
    kvattn = _kv()
    sizes = [1] * 300
    c = Case(23, sizes, 40000, 40000, "f32", history=20, bias=4)
    long = np.zeros((300, 32768), dtype=np.int32)
    long[:, :20] = c.rules["history"]
    c.rules.update(history=long, max_history=32768)
    r = np.random.RandomState(1)
    for b in (0, 150, 299):                              # some are as long as they can be
        long[b] = r.randint(0, 40000, 32768)
        c.rules["history_len"][b], c.rules["prompt_len"][b] = 32768, 10000
    c.check(dev)
    with pytest.raises(kvattn.KvAttnError) as e:
        _same(c, dev, workspace=None)
    assert e.value.status == kvattn.ERR_LDS
    x = torch.zeros((300, 40000), device=dev)
    rules = kvattn.LogitRules(**{k: _dev(v, dev) if isinstance(v, np.ndarray) else v for k, v in c.rules.items()})
    with pytest.raises(kvattn.KvAttnError) as e:
        kvattn.process_logits(x, x, rules, None, 300, 300, 40000)
    assert e.value.status == kvattn.ERR_LDS


def test_in_place_where_slices_wait_in_vain(dev):
    """Outputs in the logits' place: no slice reads another's."""
    import torch
    kvattn = _kv()
    x = torch.randn(3, 50257, device=dev)
    rules = kvattn.LogitRules(temperature=torch.ones(3, device=dev))
    want = torch.empty_like(x)
    kvattn.process_logits(want, x, kvattn.LogitRules(temperature=torch.ones(3, device=dev), workspace=None), None, 3, 3, 50257)
    before = kvattn.set_merge_poll_limit(0)
    try:
        kvattn.process_logits(x, x, rules, None, 3, 3, 50257)
        torch.cuda.synchronize()
    finally:
        kvattn.set_merge_poll_limit(before)
    assert torch.equal(x, want)


def test_captured_and_on_another_stream(dev):
    """One workspace in a graph and in eager calls between its replays, ordered."""
    import torch
    c = Case(24, [4, 4], 50257, 50257, "f32", history=100, grammar=True)
    kvattn = _kv()
    x = torch.from_numpy(c.x).to(dev)
    rules = kvattn.LogitRules(**{k: _dev(v, dev) if isinstance(v, np.ndarray) else v for k, v in c.rules.items()})
    start = _dev(c.start, dev)
    out, eager = torch.zeros_like(x), torch.zeros_like(x)
    call = lambda o: kvattn.process_logits(o, x, rules, start, 2, 8, 50257)      # noqa: E731
    call(eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
        call(out)
    side = torch.cuda.Stream()
    for _ in range(4):
        out.zero_()
        graph.replay()
        assert torch.equal(out, eager)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = torch.zeros_like(x)
            call(again)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(again, eager)


@pytest.mark.parametrize("rows,bias", [(64, 0), (64, 40), (20, 5), (300, 0)])
def test_histories_of_thousands(dev, rows, bias):
    c = Case(25, [rows - 3, 3], 33001, 33004, "f32", history=5000, bias=bias, grammar=rows == 64)
    c.check(dev)
    c.check(dev, "bf16", probs=False)


@pytest.mark.parametrize("V", [900, 50257])
def test_temperatures_whose_quotients_end(dev, V):
    """Temperatures so small or large that 1 / T is infinite or zero: the largest share, all share."""
    import torch
    kvattn = _kv()
    T = [1e-44, 1e-39, 3e38, float("inf")]
    x = torch.randn(4, V, device=dev)
    x[:, 7] = x[:, 80] = 9.0
    x[:, 3] = 20.0                                       # is forbidden
    allowed = torch.full((1, (V + 31) // 32), -1, dtype=torch.int32, device=dev)
    allowed[0, 0] = ~(1 << 3)
    rules = kvattn.LogitRules(temperature=torch.tensor(T, device=dev), allowed=allowed, num_allowed=1, allowed_stride=allowed.shape[1],
                              allowed_of=torch.zeros(4, dtype=torch.int32, device=dev))
    out = torch.full_like(x, -1.0)
    kvattn.process_logits(out, x, rules, None, 4, 4, V)
    want = torch.zeros_like(x)
    want[:2, 7] = want[:2, 80] = 0.5
    want[2:] = 1.0 / (V - 1)
    want[2:, 3] = 0.0
    # (Weights of one and their sums are whole: a quotient and a product round.)
    assert ((out - want).abs() <= 2.0 ** -20 * want).all()


@pytest.mark.parametrize("starts", [True, False])
def test_bits_behind_the_last_row(dev, starts):
    """Masks with bits of tokens that the sequence does not have."""
    import torch
    kvattn = _kv()
    start = np.array([0, 3, 3, 5, 8] if starts else range(9), dtype=np.int32)
    x = torch.full((8, 1000), 4.0, device=dev)
    rules = kvattn.LogitRules(tokens=torch.arange(100, 108, dtype=torch.int32, device=dev), mask_words=2,
                              masks=torch.full((8, 2), -1, dtype=torch.int64, device=dev),
                              presence=torch.full((len(start) - 1,), 1.0, device=dev))
    out = torch.zeros_like(x)
    kvattn.process_logits(out, x, rules, _dev(start, dev) if starts else None, len(start) - 1, 8, 1000, probs=False)
    want = torch.full_like(x, 4.0)
    for lo, hi in zip(start[:-1].tolist(), start[1:].tolist()):
        want[lo:hi, 100 + lo:100 + hi] = 3.0
    assert torch.equal(out, want)


@pytest.mark.parametrize("rows,history,bias", [(120, 20000, 0), (120, 20000, 30), (90, 9000, 0), (100, 3, 17000), (250, 12000, 0)])
def test_tables_of_many_ids(dev, rows, history, bias):
    c = Case(26, [1] * rows, 33001, 33004, "f32", history=20, bias=4)
    r = np.random.RandomState(2)
    long = np.zeros((rows, history), dtype=np.int32)
    for b in (0, rows // 2, rows - 1):
        long[b] = r.randint(0, 33001, history)
        c.rules["history_len"][b], c.rules["prompt_len"][b] = history, history // 3
    for b in range(rows):
        c.rules["history_len"][b] = min(c.rules["history_len"][b], history)
        if b not in (0, rows // 2, rows - 1):
            long[b, :min(20, history)] = c.rules["history"][b, :min(20, history)]
    c.rules.update(history=long, max_history=history)
    if bias:                                             # one sequence has nearly all of them
        n = int(c.rules["bias_start"][-1])
        ids = np.concatenate([c.rules["bias_ids"][:n], r.permutation(33001)[:bias - 5]]).astype(np.int32)
        c.rules["bias_start"][-1] = len(ids)
        c.rules.update(bias_ids=ids, bias=r.standard_normal(len(ids)).astype(np.float32), num_bias=len(ids), max_bias=bias)
    c.check(dev)
