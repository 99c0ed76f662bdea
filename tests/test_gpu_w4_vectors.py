"""Fully connected layers on 4-bit weights for very many vectors, against treeref.w4_layer."""
import numpy as np
import pytest

import treeref
from test_gpu_w4 import _pack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["int4", "fp4"])
@pytest.mark.parametrize("pre", [False, True])
def test_more_vectors_than_a_grid_has_columns(dev, kind, pre):
    """65535 columns of 64 vectors and some more: vectors on both sides of the border."""
    import torch
    from cuda_gpt2_inference_amd import kvattn
    M, K, group, edge = 20, 32, 32, 65535 * 64
    B = edge + 77
    r = np.random.RandomState(3)
    nib = r.randint(0, 16, (M, K)).astype(np.uint8)
    scale = treeref.bf16(np.exp(r.standard_normal((M, 1))) * 0.1)
    bias = treeref.bf16(r.standard_normal(M))
    w4 = kvattn.w4_pack(torch.from_numpy(_pack(nib)).to(dev), torch.from_numpy(scale).to(torch.bfloat16).to(dev), M, K, group, w_dtype=kind)
    some = treeref.bf16(r.standard_normal((1000, K)))
    x = torch.from_numpy(some).to(torch.bfloat16).to(dev).repeat(B // 1000 + 1, 1)[:B].contiguous()
    out = torch.full((B + 1, M), 33.0, device=dev)
    before = torch.full((B + 1, M), 33.0, device=dev) if pre else None
    kvattn.gemv_w4(out, w4, x, B, M, K, group=group, w_dtype=kind, out_dtype="f32", pre_gelu=before,
                   bias=torch.from_numpy(bias).to(torch.bfloat16).to(dev))
    ref, err = treeref.w4_layer(nib, scale, some.astype(np.float64), bias.astype(np.float64), kind)
    err = err + 2.0 ** -24 * np.abs(ref)
    for got in (out,) + ((before,) if pre else ()):
        assert (got[B] == 33.0).all()
        first = got[:1000].double().cpu().numpy()
        assert (np.abs(first - ref) <= err).all()
        # A vector's outputs are the same wherever it stands.
        again = got[:1000].repeat(B // 1000 + 1, 1)[:B]
        assert torch.equal(got[:B], again)
