"""gemv_w4's documented limits, without a GPU: what a launch could not hold is refused as a shape."""
import pytest

A = 1 << 20          # an aligned address that no refused call looks at


@pytest.mark.parametrize("M,K,group", [((1 << 28) - 31, 1152, 128), ((1 << 28) - 1, 1088, 64), ((1 << 28) - 31, 64, 64)])
def test_more_rows_than_a_grid_holds(M, K, group):
    from cuda_gpt2_inference_amd import kvattn
    assert kvattn.lib().kvattn_gemv_w4(A, None, A, A, None, 1, M, K, group, 4, 1, 0, None) == kvattn.ERR_SHAPE
