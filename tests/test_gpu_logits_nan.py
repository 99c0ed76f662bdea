"""Probabilities of rows with NaN and infinities that are allowed, wherever in the row they stand and however it is cut into
slices: NaN where a token weighs anything, zero elsewhere."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def _kv():
    from cuda_gpt2_inference_amd import kvattn
    return kvattn


def _call(dev, x, keep, T, dtype="f32", probs=True, **extra):
    """The probabilities of rows x (numpy) of which the tokens `keep` (bool) are allowed."""
    import torch
    kvattn = _kv()
    rows, V = x.shape
    words = (V + 31) // 32
    bits = np.zeros((rows, 32 * words), dtype=np.uint64)
    bits[:, :V] = keep
    line = (bits.reshape(rows, words, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32).view(np.int32)
    td = torch.float32 if dtype == "f32" else torch.bfloat16
    rules = kvattn.LogitRules(allowed=torch.from_numpy(line).to(dev), num_allowed=rows, allowed_stride=words,
                              temperature=torch.full((rows,), T, device=dev), **extra)
    xd = torch.from_numpy(x).to(dev).to(td)
    out = torch.full((rows, V), 9.0, dtype=td, device=dev)
    kvattn.process_logits(out, xd, rules, None, rows, rows, V, dtype=dtype, probs=probs)
    return out.float().cpu().numpy()


# (V, rows, workspace): slices of every size, one workgroup a row with the row in registers, and read in every pass.
SHAPES = [(700, 4, True), (50257, 4, True), (50257, 30, True), (50257, 70, True), (50257, 140, True), (50257, 4, False), (3001, 300, True),
          (60000, 4, False), (60000, 200, True)]


@pytest.mark.parametrize("V,rows,workspace", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_nan_alone_in_its_slice(dev, V, rows, workspace, dtype):
    extra = {} if workspace else dict(workspace=None)
    r = np.random.RandomState(V + rows)
    x = np.full((rows, V), 100.0, dtype=np.float32)
    keep = np.zeros((rows, V), dtype=bool)
    want = np.zeros((rows, V), dtype=np.float32)
    for t in range(rows):
        tokens = r.permutation(V)[:4]
        x[t, tokens] = r.standard_normal(4)
        x[t, tokens[0]] = NAN
        kind = t % 4                     # 0: numbers and a NaN; 1: the NaN alone; 2: NaN beside an allowed -inf; 3: no NaN
        keep[t, tokens[1:] if kind == 3 else tokens[:1] if kind == 1 else tokens] = True
        if kind == 2:
            x[t, tokens[1:]] = -INF
        if kind == 3:
            w = np.exp(x[t, tokens[1:]].astype(np.float64) / 0.8)
            want[t, tokens[1:]] = w / w.sum()
        else:
            want[t, tokens[:1] if kind else tokens] = NAN
    got = _call(dev, x, keep, 0.8, dtype, **extra)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    # bf16: the logit is rounded (an exponent of at most 5 / 0.8 by 2^-8 of it) and so is the result.
    assert (np.abs(got - want)[~np.isnan(want)] <= (1e-5 if dtype == "f32" else 0.06) * want[~np.isnan(want)]).all()


@pytest.mark.parametrize("V,rows,workspace", SHAPES)
def test_an_infinity_takes_all(dev, V, rows, workspace):
    """Beside +inf every other token weighs nothing, in its slice and in others."""
    extra = {} if workspace else dict(workspace=None)
    r = np.random.RandomState(V)
    x = r.standard_normal((rows, V)).astype(np.float32)
    at = r.randint(0, V, rows)
    x[np.arange(rows), at] = INF
    got = _call(dev, x, np.ones((rows, V), dtype=bool), 0.8, **extra)
    want = np.zeros((rows, V), dtype=np.float32)
    want[np.arange(rows), at] = NAN
    assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("V,rows,workspace", SHAPES)
def test_the_likeliest_among_numbers(dev, V, rows, workspace):
    extra = {} if workspace else dict(workspace=None)
    r = np.random.RandomState(V + 1)
    x = r.standard_normal((rows, V)).astype(np.float32)
    x[:, ::3] = NAN
    keep = r.rand(rows, V) < 0.5
    x[1] = NAN                                           # no number: zeros
    keep[2] = False
    want = np.zeros((rows, V), dtype=np.float32)
    for t in range(rows):
        y = np.where(keep[t] & ~np.isnan(x[t]), x[t], -INF)
        if y.max() > -INF:
            want[t, int(np.argmax(y))] = 1.0
    assert np.array_equal(_call(dev, x, keep, 0.0, **extra), want)


@pytest.mark.parametrize("V", [3001, 50257])
def test_slices_that_wait_in_vain(dev, V):
    """The same where every slice works the others out."""
    import torch
    kvattn = _kv()
    r = np.random.RandomState(5)
    x = r.standard_normal((6, V)).astype(np.float32)
    keep = np.zeros((6, V), dtype=bool)
    keep[:, 5] = keep[:, V - 5] = True
    keep[3:] = True
    x[:3, V - 5], x[1, 5], x[2, 5], x[3, 7], x[4, V - 9] = NAN, NAN, -INF, INF, NAN
    want = _call(dev, x, keep, 0.7)
    before = kvattn.set_merge_poll_limit(0)
    try:
        got = _call(dev, x, keep, 0.7)
        torch.cuda.synchronize()
    finally:
        kvattn.set_merge_poll_limit(before)
    assert np.array_equal(got, want, equal_nan=True) and np.isnan(got[:3, V - 5]).all() and np.isnan(got[0, 5])
