"""Rules on logits at the documented limits."""
import pytest

pytestmark = pytest.mark.gpu


def test_logits_of_as_many_rows_as_there_may_be(dev):
    """2^21 rows of which each is four slices: 2^32 threads are more than one launch takes."""
    import torch
    from cuda_gpt2_inference_amd import kvattn
    rows, V = 1 << 21, 3 * 4096 + 4
    x = torch.zeros((rows, V), dtype=torch.bfloat16, device=dev)         # 52 GB, in place
    split = 2 * rows // 3 + 1
    start = torch.tensor([0, split, rows], dtype=torch.int32, device=dev)
    rules = kvattn.LogitRules(bias_start=torch.tensor([0, 2, 4], dtype=torch.int32, device=dev), num_bias=4, max_bias=2,
                              bias_ids=torch.tensor([5, V - 1, 4096, 8191], dtype=torch.int32, device=dev),
                              bias=torch.tensor([1.0, 2.0, 3.0, 4.0], device=dev))
    kvattn.process_logits(x, x, rules, start, 2, rows, V, dtype="bf16", probs=False)
    assert (x[:split, 5] == 1).all() and (x[:split, V - 1] == 2).all()
    assert (x[split:, 4096] == 3).all() and (x[split:, 8191] == 4).all()
    step = rows // 32
    assert sum(int((x[r:r + step] != 0).sum()) for r in range(0, rows, step)) == 2 * rows
