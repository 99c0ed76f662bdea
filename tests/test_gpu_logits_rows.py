"""Probabilities of rows that one workgroup reads again in every pass: vocabularies that do not fit its registers, where
there is no workspace, where the outputs take the logits' place, or where there are more rows than slices run at once."""
import numpy as np
import pytest

from test_gpu_logits import Case, _dev, _kv

pytestmark = pytest.mark.gpu

BIG = 1 << 18


def _case(seed, sizes, V, stride, dtype, **kw):
    rules = dict(history=300, bias=20, grammar=True, branches=True)
    rules.update(kw)
    return Case(seed, sizes, V, stride, dtype, **rules)


@pytest.mark.parametrize("V,stride", [(60000, 60000), (53249, 53250), (BIG - 3, BIG), (BIG, BIG)])
@pytest.mark.parametrize("dtype,out_dtype", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
def test_without_a_workspace(dev, V, stride, dtype, out_dtype):
    c = _case(31, [2, 0, 3], V, stride, dtype)
    c.rules["workspace"] = None
    c.check(dev, out_dtype)
    c.rules["temperature"][:] = 0.0
    c.check(dev, out_dtype)


@pytest.mark.parametrize("kw", [dict(history=0, bias=0, grammar=False, branches=False, penalties=False), dict(grammar=False),
                                dict(history=0, branches=False, bias=0), dict(history=4000, wide_ids=True), dict(temperature=False)])
def test_each_rule(dev, kw):
    c = _case(32, [3, 1], 60000, 60003, "f32", **kw)
    c.rules["workspace"] = None
    c.check(dev, offset=1, out_stride=60001)


@pytest.mark.parametrize("V", [60000, 60001, BIG])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place(dev, V, dtype):
    """The same bits as beside the logits without a workspace."""
    import torch
    kvattn = _kv()
    c = _case(33, [2, 1, 1], V, V + 3, dtype)
    c.x = np.nan_to_num(c.x)
    td = torch.float32 if dtype == "f32" else torch.bfloat16
    x = torch.from_numpy(c.x).to(td).to(dev)
    rules = {k: _dev(v, dev) if isinstance(v, np.ndarray) else v for k, v in c.rules.items()}
    c.rules["workspace"] = None
    want = c.run(dev, dtype, True)
    c.check(dev, dtype)
    kvattn.process_logits(x, x, kvattn.LogitRules(**rules), _dev(c.start, dev), c.B, c.N, V, row_stride=V + 3, out_stride=V + 3, dtype=dtype)
    assert np.array_equal(x[:, :V].double().cpu().numpy(), want)
    assert (x[:, V:] == 0).all()


@pytest.mark.parametrize("rows,V", [(171, 60000), (52, BIG)])
def test_more_rows_than_slices_run_at_once(dev, rows, V):
    c = _case(34, [rows - 3, 3], V, V, "bf16", history=100)
    c.check(dev, "f32")


def test_captured(dev):
    """Replays against the eager result, the logits new every time."""
    import torch
    kvattn = _kv()
    V = 60000
    c = _case(35, [2, 2], V, V, "f32")
    rules = kvattn.LogitRules(**{k: _dev(v, dev) if isinstance(v, np.ndarray) else v for k, v in c.rules.items()}, workspace=None)
    start = _dev(c.start, dev)
    source = torch.from_numpy(c.x).to(dev)
    x, eager = source.clone(), source.clone()
    call = lambda y: kvattn.process_logits(y, y, rules, start, 2, 4, V)      # noqa: E731
    call(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(x)
    for step in range(4):
        shifted = source + step
        x.copy_(shifted)
        graph.replay()
        eager = shifted.clone()
        call(eager)
        torch.cuda.synchronize()
        assert torch.equal(x, eager)
