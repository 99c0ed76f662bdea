"""Fully connected layers on 4-bit weights with group scales, against treeref.w4_layer in 64 bits."""
import numpy as np
import pytest

import treeref

pytestmark = pytest.mark.gpu


def _kv():
    from cuda_gpt2_inference_amd import kvattn
    return kvattn


def _pack(nib):
    return (nib[:, 0::2] | (nib[:, 1::2] << 4)).astype(np.uint8)


class Layer:
    def __init__(self, dev, kind, B, M, K, group, seed=0):
        import torch
        r = np.random.RandomState(seed + M + K)
        self.dev, self.kind, self.B, self.M, self.K, self.group = dev, kind, B, M, K, group
        self.nib = r.randint(0, 16, (M, K)).astype(np.uint8)              # every code, -8 among INT4's
        self.scale = treeref.bf16(np.exp(r.standard_normal((M, K // group))) * 0.02)
        self.x = treeref.bf16(r.standard_normal((B, K)))
        self.bias = treeref.bf16(r.standard_normal(M))
        self.w4 = _kv().w4_pack(torch.from_numpy(_pack(self.nib)).to(dev), torch.from_numpy(self.scale).to(torch.bfloat16).to(dev),
                                M, K, group, w_dtype=kind)

    def run(self, out_dtype="bf16", gelu=False, pre=False, bias=True, x=None):
        import torch
        td = torch.float32 if out_dtype == "f32" else torch.bfloat16
        out = torch.full((self.B + 1, self.M), 33.0, dtype=td, device=self.dev)
        pre_gelu = torch.full((self.B + 1, self.M), 33.0, dtype=td, device=self.dev) if pre else None
        xd = torch.from_numpy(self.x if x is None else x).to(torch.bfloat16).to(self.dev)
        _kv().gemv_w4(out, self.w4, xd, self.B, self.M, self.K, group=self.group, w_dtype=self.kind, out_dtype=out_dtype, gelu=gelu,
                      pre_gelu=pre_gelu, bias=torch.from_numpy(self.bias).to(torch.bfloat16).to(self.dev) if bias else None)
        assert (out[self.B] == 33.0).all() and (pre_gelu is None or (pre_gelu[self.B] == 33.0).all())
        return out[:self.B].double().cpu().numpy(), None if pre_gelu is None else pre_gelu[:self.B].double().cpu().numpy()

    def check(self, out_dtype="bf16", gelu=False, pre=False, bias=True):
        got, got_pre = self.run(out_dtype, gelu, pre, bias)
        ref, err = treeref.w4_layer(self.nib, self.scale, self.x.astype(np.float64), self.bias.astype(np.float64) * bias, self.kind)
        half = treeref.HALF_STEP[out_dtype]
        if pre:
            assert (np.abs(got_pre - ref) <= err + half * np.abs(ref) + 2.0 ** -126).all()
        if gelu:
            # GELU's slope is at most 1.13; its tanh, cube and products are a few float roundings of what they are.
            ref, err = treeref.gelu(ref), 1.13 * err + 16 * 2.0 ** -24 * (np.abs(ref) + np.abs(ref) ** 3 * (np.abs(ref) < 6))
        bad = np.abs(got - ref) > err + half * np.abs(ref) + 2.0 ** -126
        assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], ref[bad][:4])


@pytest.mark.parametrize("kind", ["int4", "fp4"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("B,M,K", [(1, 1, 128), (1, 1024, 1024), (2, 15, 384), (3, 17, 1664), (16, 40, 256), (17, 100, 640),
                                   (33, 33, 1280), (64, 257, 768), (65, 48, 128), (130, 20, 2048), (1, 50304, 768)])
def test_layers(dev, kind, group, B, M, K):
    Layer(dev, kind, B, M, K, group).check("f32")


@pytest.mark.parametrize("kind", ["int4", "fp4"])
@pytest.mark.parametrize("B,M,K,group", [(1, 70, 32, 32), (5, 64, 96, 32), (40, 30, 1600, 64), (2, 500, 320, 64), (9, 100, 6400, 32),
                                         (70, 2000, 64, 64)])
def test_rows_that_end_inside_a_block(dev, kind, B, M, K, group):
    Layer(dev, kind, B, M, K, group).check("f32")


@pytest.mark.parametrize("kind,group", [("int4", 64), ("fp4", 32), ("int4", 128)])
@pytest.mark.parametrize("B,M,K", [(4, 9001, 1280), (1, 40007, 640), (7, 5200, 256), (16, 39000, 256), (26, 6400, 512), (20, 12000, 256),
                                   (30, 20011, 384), (64, 4115, 256), (64, 9000, 256), (40, 24601, 1408), (130, 4100, 256),
                                   (100, 16400, 256)])
def test_tall(dev, kind, group, B, M, K):
    """Each way of tiling, rows that end inside a tile."""
    Layer(dev, kind, B, M, K, group).check("f32")


@pytest.mark.parametrize("kind", ["int4", "fp4"])
@pytest.mark.parametrize("B", [1, 26, 70])
@pytest.mark.parametrize("kw", [dict(), dict(gelu=True), dict(gelu=True, pre=True), dict(bias=False), dict(pre=True),
                                dict(out_dtype="f32", gelu=True, pre=True)])
def test_epilogue(dev, kind, B, kw):
    Layer(dev, kind, B, 203, 512, 64).check(**kw)


@pytest.mark.parametrize("kind", ["int4", "fp4"])
@pytest.mark.parametrize("B", [3, 40])
def test_a_vector_that_is_not_finite(dev, kind, B):
    """A vector's NaN and infinities stay its own."""
    c = Layer(dev, kind, B, 100, 320, 32)
    want, _ = c.run("f32")
    x = c.x.copy()
    x[1, 5], x[1, 300] = np.nan, np.inf
    got, _ = c.run("f32", x=x)
    keep = np.arange(B) != 1
    assert np.array_equal(got[keep], want[keep]) and not np.isfinite(got[1]).all()


@pytest.mark.parametrize("kind", ["int4", "fp4"])
@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("M,K,group", [(5, 64, 32), (40, 1600, 64), (17, 384, 128)])
def test_quantize(dev, kind, src, M, K, group):
    """The same bytes as the codes and scales laid out: ties, zero groups, NaN and infinities among them."""
    import torch
    kvattn = _kv()
    r = np.random.RandomState(M)
    W = r.standard_normal((M, K)).astype(np.float32)
    W[0, :group] = 0.0
    W[1, :group] = np.resize([7.0, 0.5, -1.5, 2.5, -3.5, 0.25, 0.75, -0.0, 1.25, 5.0, 6.0, 1e-30], group)
    W[2, 3], W[3, 3], W[4, 3] = np.nan, np.inf, 1e-39
    if src == "bf16":
        W = treeref.bf16(W)
    nib, scale = treeref.w4_codes(W, group, kind)
    td = torch.float32 if src == "f32" else torch.bfloat16
    got = kvattn.w4_quantize(torch.from_numpy(W).to(td).to(dev), M, K, group, w_dtype=kind, src_dtype=src,
                             out=torch.zeros(kvattn.w4_bytes(M, K, group), dtype=torch.uint8, device=dev))
    want = kvattn.w4_pack(torch.from_numpy(_pack(nib)).to(dev), torch.from_numpy(scale).to(torch.bfloat16).to(dev), M, K, group,
                          w_dtype=kind, out=torch.zeros_like(got))
    assert torch.equal(got, want)


def test_scales_of_any_size(dev):
    """Scales of zero, and far apart within a row."""
    c = Layer(dev, "int4", 4, 32, 256, 32)
    import torch
    r = np.random.RandomState(1)
    c.scale = treeref.bf16(np.exp2(r.randint(-60, 60, c.scale.shape).astype(np.float32)) * (r.rand(*c.scale.shape) < 0.8))
    c.w4 = _kv().w4_pack(torch.from_numpy(_pack(c.nib)).to(dev), torch.from_numpy(c.scale).to(torch.bfloat16).to(dev), 32, 256, 32, w_dtype="int4")
    c.check("f32")
