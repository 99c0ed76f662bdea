"""What the entry points for trees of drafted tokens, rules on logits and 4-bit weights refuse, without a GPU."""
import ctypes

import pytest

A = 1 << 20          # an aligned address that no refused call looks at


def _kv():
    from cuda_gpt2_inference_amd import kvattn
    return kvattn


def _status(name, args, **kw):
    """The entry point's status with some arguments replaced."""
    names = list(args)
    values = {**args, **kw}
    assert set(kw) <= set(names)
    return getattr(_kv().lib(), name)(*[values[k] for k in names])


TREE = dict(out=A, qkv=A, pages=A, scales=None, table=A, max_pages=4, page_rows=64, num_pages=8, start=A, lens=A, masks=A,
            mask_words=1, B=2, num_tokens=8, max_new=8, NH=2, hs=64, ws=None, ws_bytes=0, S=1, kv=1, stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(hs=32), 3), (dict(B=0), 4), (dict(NH=0), 4), (dict(num_tokens=0), 4), (dict(max_new=0), 4), (dict(mask_words=0), 4),
    (dict(mask_words=5), 4), (dict(max_new=65, num_tokens=65), 4), (dict(page_rows=63), 4), (dict(page_rows=0), 4),
    (dict(max_pages=0), 4), (dict(B=65536, NH=1), 4), (dict(num_tokens=1 << 24, NH=2), 4), (dict(kv=6), 5), (dict(kv=-1), 5),
    (dict(kv=2), 5), (dict(kv=4), 5), (dict(kv=5), 5), (dict(out=None), 1), (dict(qkv=None), 1), (dict(pages=None), 1),
    (dict(table=None), 1), (dict(start=None), 1), (dict(lens=None), 1), (dict(masks=None), 1), (dict(masks=A + 4), 2),
    (dict(qkv=A + 8), 2), (dict(out=A + 8), 2), (dict(pages=A + 8), 2), (dict(start=A + 2), 2), (dict(lens=A + 2), 2),
    (dict(kv=3, scales=A + 2), 2), (dict(S=-100), 8), (dict(S=70000), 8), (dict(S=2), 7), (dict(S=2, ws=A + 8, ws_bytes=1 << 20), 2),
    (dict(S=2, ws=A, ws_bytes=64), 7)])
def test_decode_tree(kw, status):
    assert _status("kvattn_paged_decode_tree", TREE, **kw) == status


MASKS = dict(masks=A, positions=A, parents=A, start=A, lens=A, B=1, num_tokens=4, words=1, stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(B=0), 4), (dict(B=(1 << 20) + 1), 4), (dict(num_tokens=-1), 4), (dict(words=0), 4), (dict(words=5), 4), (dict(num_tokens=(1 << 30) + 1), 4),
    (dict(masks=None), 1), (dict(parents=None), 1), (dict(start=None), 1), (dict(lens=None), 1), (dict(masks=A + 4), 2),
    (dict(parents=A + 1), 2), (dict(positions=A + 2), 2), (dict(num_tokens=0, masks=None, parents=None, start=None), 0)])
def test_tree_masks(kw, status):
    assert _status("kvattn_tree_masks", MASKS, **kw) == status


KEEP = dict(pages=A, scales=A, page_rows=64, num_pages=4, slots=A, path=A, start=A, B=1, num_tokens=4, NH=2, hs=64, kv=1, stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(hs=128), 3), (dict(B=0), 4), (dict(NH=0), 4), (dict(page_rows=0), 4), (dict(num_pages=0), 4), (dict(num_tokens=-1), 4),
    (dict(B=1 << 20, NH=1 << 10), 4), (dict(kv=6), 5), (dict(kv=2, scales=None), 5), (dict(pages=None), 1), (dict(slots=None), 1),
    (dict(path=None), 1), (dict(start=None), 1), (dict(pages=A + 8), 2), (dict(slots=A + 4), 2), (dict(path=A + 2), 2),
    (dict(num_tokens=0, pages=None), 0)])
def test_keep(kw, status):
    assert _status("kvattn_paged_keep", KEEP, **kw) == status


VERIFY = dict(tokens=A, path=A, counts=A, kept=A, p=A, tree=A, parents=A, u=A, draw=A, start=A, lens=A, B=1, num_tokens=4, V=100,
              row=100, dtype=0, ws=A, ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(B=0), 4), (dict(B=65537), 4), (dict(V=0), 4), (dict(V=(1 << 24) + 1, row=1 << 25), 4), (dict(row=99), 4),
    (dict(num_tokens=-1), 4), (dict(dtype=2), 5), (dict(counts=None), 1), (dict(start=None), 1), (dict(lens=None), 1),
    (dict(tokens=None), 1), (dict(path=None), 1), (dict(p=None), 1), (dict(tree=None), 1), (dict(parents=None), 1),
    (dict(u=None), 1), (dict(draw=None), 1), (dict(ws=None), 7), (dict(ws_bytes=16), 7), (dict(ws=A + 16), 2), (dict(p=A + 2), 2),
    (dict(path=A + 2), 2), (dict(kept=A + 1), 2), (dict(draw=A + 3), 2)])
def test_verify_tree(kw, status):
    assert _status("kvattn_verify_tree", VERIFY, **kw) == status


LOGITS = dict(out=A, x=A, rules=None, start=A, B=2, rows=4, V=100, row=100, out_row=100, dtype=0, out_dtype=0, probs=1, stream=None)


@pytest.mark.parametrize("kw,rules,status", [
    (dict(dtype=2), {}, 5), (dict(out_dtype=3), {}, 5), (dict(B=0), {}, 4), (dict(rows=-1), {}, 4), (dict(rows=(1 << 21) + 1), {}, 4),
    (dict(V=0), {}, 4), (dict(V=(1 << 18) + 1, row=1 << 19, out_row=1 << 19), {}, 4), (dict(row=99), {}, 4), (dict(out_row=99), {}, 4),
    (dict(start=None), {}, 4), (dict(out=None), {}, 1), (dict(x=None), {}, 1), (dict(x=A + 2), {}, 2), (dict(start=A + 2), {}, 2),
    (dict(rows=0, x=None, out=None), {}, 0),
    ({}, dict(history=A, history_len=A, max_history=0), 4), ({}, dict(history=A, history_len=A, max_history=32769), 4),
    ({}, dict(history=A, max_history=5), 1), ({}, dict(tokens=A, mask_words=1), 1), ({}, dict(masks=A, mask_words=1), 1),
    ({}, dict(tokens=A, masks=A, mask_words=5), 4), ({}, dict(tokens=A, masks=A + 4, mask_words=1), 2),
    ({}, dict(bias_start=A, num_bias=-1, max_bias=1), 4), ({}, dict(bias_start=A, num_bias=3, max_bias=3, bias_ids=A), 1),
    ({}, dict(bias_start=A, num_bias=3, max_bias=40000, bias_ids=A, bias=A), 4),
    ({}, dict(allowed=A, num_allowed=0, allowed_stride=4), 4), ({}, dict(allowed=A, num_allowed=2, allowed_stride=3), 4),
    ({}, dict(temperature=A + 1), 2), ({}, dict(repetition=A + 2), 2),
    ({}, dict(workspace=A, workspace_bytes=64), 7), ({}, dict(workspace=A + 4, workspace_bytes=1 << 20), 2),
    (dict(V=1 << 18, row=1 << 18, out_row=1 << 18), dict(history=A, history_len=A, max_history=32768, bias_start=A, bias_ids=A, bias=A,
                                                         num_bias=32768, max_bias=32768), 10)])
def test_process_logits(kw, rules, status):
    kvattn = _kv()
    if rules:
        kw = dict(kw, rules=kvattn.LogitRules(**rules).address)
        keep = kvattn.LogitRules(**rules)
        kw["rules"] = keep.address
    assert _status("kvattn_process_logits", LOGITS, **kw) == status


def test_logit_rules_of_no_such_name():
    with pytest.raises(TypeError):
        _kv().LogitRules(histroy=A)
    assert ctypes.sizeof(_kv()._LogitRules) == 14 * 8 + 6 * 4 + 16


GEMV = dict(out=A, pre=None, w4=A, x=A, bias=None, B=1, M=10, K=256, group=64, w=4, out_dtype=1, gelu=0, stream=None)


@pytest.mark.parametrize("kw,status", [
    (dict(M=1 << 28, K=1024), 4), (dict(w=1), 5), (dict(w=6), 5), (dict(out_dtype=2), 5), (dict(group=16), 4), (dict(group=256), 4), (dict(K=250), 4),
    (dict(K=32, group=64), 4), (dict(M=0), 4), (dict(B=0), 4), (dict(K=(1 << 20) + 64), 4), (dict(B=1 << 20, M=1 << 12), 4),
    (dict(out=None), 1), (dict(w4=None), 1), (dict(x=None), 1), (dict(w4=A + 8), 2), (dict(x=A + 2), 2), (dict(out=A + 1), 2),
    (dict(bias=A + 1), 2), (dict(pre=A + 2, out_dtype=0), 2)])
def test_gemv_w4(kw, status):
    assert _status("kvattn_gemv_w4", GEMV, **kw) == status


def test_w4_layout_calls():
    kvattn = _kv()
    lib = kvattn.lib()
    assert kvattn.w4_bytes(16, 128, 128) == 1024 + 32 and kvattn.w4_bytes(17, 129 * 32, 32) == 2 * 33 * (1024 + 128)
    assert kvattn.w4_bytes(16, 100, 32) == 0 and kvattn.w4_bytes(16, 128, 48) == 0 and kvattn.w4_bytes(0, 128, 32) == 0
    assert lib.kvattn_w4_pack(A, A, A, 16, 128, 32, 2, None) == kvattn.ERR_DTYPE
    assert lib.kvattn_w4_pack(A, A, A, 16, 100, 32, 4, None) == kvattn.ERR_SHAPE
    assert lib.kvattn_w4_pack(A, None, A, 16, 128, 32, 4, None) == kvattn.ERR_NULL_POINTER
    assert lib.kvattn_w4_pack(A, A + 4, A, 16, 128, 32, 4, None) == kvattn.ERR_MISALIGNED
    assert lib.kvattn_w4_quantize(A, A, 16, 128, 32, 2, 4, None) == kvattn.ERR_DTYPE
    assert lib.kvattn_w4_quantize(A, A, 16, 128, 32, 0, 1, None) == kvattn.ERR_DTYPE
    assert lib.kvattn_w4_quantize(A, None, 16, 128, 32, 0, 4, None) == kvattn.ERR_NULL_POINTER
    assert lib.kvattn_w4_quantize(A + 1, A, 16, 128, 32, 0, 4, None) == kvattn.ERR_MISALIGNED
