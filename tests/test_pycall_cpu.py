"""The binding's calls by address (_pycall.Call) against ctypes: arguments of every kind and width."""
import ctypes

import numpy as np
import pytest

ALIGNED = 1 << 20


def _kv():
    from cuda_gpt2_inference_amd import kvattn
    kvattn.lib()
    return kvattn


def _call(fn, words):
    from cuda_gpt2_inference_amd._pycall import Call
    return Call(ctypes.cast(fn, ctypes.c_void_p).value, words)


_W = ctypes.c_longlong


def test_words_arrive():
    """Sums that only come out if every word is in its place, in registers and on the stack."""
    got = []

    def seen(*words):
        got[:] = words
        return 7
    for n in (0, 1, 5, 6, 7, 16, 17, 21, 24):
        fn = ctypes.CFUNCTYPE(ctypes.c_int, *[_W] * n)(seen)
        args = [(i + 1) * 0x0123456789AB for i in range(n)]
        assert _call(fn, n)(*args) == 7 and got == args


def test_kinds():
    import torch
    got = []

    def seen(*words):
        got[:] = words
        return -3
    fn = ctypes.CFUNCTYPE(ctypes.c_int, *[_W] * 6)(seen)
    call = _call(fn, 6)
    x = torch.zeros(8)
    assert call(x, None, -1, True, np.int64(5), x[2:]) == -3
    assert got == [x.data_ptr(), 0, -1, 1, 5, x.data_ptr() + 8]
    assert call(1 << 63, (1 << 64) - 1, -(1 << 63), 0, 2 ** 70 + 9, torch.nn.Parameter(x)) == -3
    assert got == [-(1 << 63), -1, -(1 << 63), 0, 9, x.data_ptr()]
    for bad in (1.5, "1", object()):
        with pytest.raises(TypeError):
            call(bad, 0, 0, 0, 0, 0)
    for args in ((), (1,) * 5, (1,) * 7):
        with pytest.raises(TypeError):
            call(*args)
    with pytest.raises(TypeError):
        call(1, 1, 1, 1, 1, w=1)


def test_narrow_parameters_read_their_own_width():
    got = []

    def seen(*words):
        got[:] = words
        return 0
    kinds = [ctypes.c_int, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_longlong] * 3
    fn = ctypes.CFUNCTYPE(ctypes.c_int, *kinds)(seen)
    _call(fn, 12)(*[-2, 2 ** 40, 2 ** 41, -5] * 3)
    assert got == [-2, 2 ** 40, 2 ** 41, -5] * 3


def test_no_call_without_an_address():
    from cuda_gpt2_inference_amd._pycall import Call
    for args in ((0, 1), (1, -1), (1, 25)):
        with pytest.raises(ValueError):
            Call(*args)


def test_refusals_are_ctypes_own():
    """The same status as through ctypes, for every entry point that the binding calls so (null pointers)."""
    kvattn = _kv()
    names = ["kvattn_cache_write", "kvattn_decode", "kvattn_append_decode", "kvattn_paged_cache_write", "kvattn_paged_decode",
             "kvattn_paged_decode_tokens", "kvattn_paged_reserve", "kvattn_paged_store", "kvattn_paged_load",
             "kvattn_verify_drafts"]
    for name in names:
        types = kvattn.SIGNATURES[name][1]
        assert len(types) <= 24 and all(t in (kvattn._vp, kvattn._i, kvattn._ll, kvattn._sz) for t in types), name
        for value in (0, 1, 64, -1):
            args = [None if t is kvattn._vp else (abs(value) if t is kvattn._sz else value) for t in types]
            want = getattr(kvattn.lib(), name)(*args)
            assert want != kvattn.OK and getattr(kvattn._call, name)(*args) == want, (name, value)


def test_wrappers_without_the_extension(monkeypatch):
    """An interpreter that the extension was not built for has ctypes."""
    import sys
    import torch
    kvattn = _kv()
    monkeypatch.setitem(sys.modules, "cuda_gpt2_inference_amd._pycall", None)
    monkeypatch.setattr(kvattn, "_call", kvattn._Calls())
    x = torch.zeros(64, dtype=torch.int32)
    cache = kvattn.PagedCache(x, x, 1, 64, 0)          # no pages: refused
    with pytest.raises(kvattn.KvAttnError) as e:
        kvattn.paged_reserve(cache, x, x, x, x, 1, lens=x, token_start=x, slot_map=x, max_tokens=1, stream=0)
    assert e.value.status == kvattn.ERR_SHAPE
    with pytest.raises(kvattn.KvAttnError) as e:
        kvattn.paged_store(cache, x, None, 1, 1, 64, kv_dtype="bf16", stream=0)
    assert e.value.status in (kvattn.ERR_SHAPE, kvattn.ERR_NULL_POINTER)


def _calls(monkeypatch, extension):
    import sys
    kvattn = _kv()
    if not extension:
        monkeypatch.setitem(sys.modules, "cuda_gpt2_inference_amd._pycall", None)
    monkeypatch.setattr(kvattn, "_call", kvattn._Calls())
    return kvattn


@pytest.mark.parametrize("extension", [True, False])
def test_integers_are_values(monkeypatch, extension):
    """Where an entry point has an integer, every argument gives what it gives through ctypes: the value of a tensor of
    one integer (never its address), and a refusal for what is no integer."""
    import torch
    kvattn = _calls(monkeypatch, extension)
    kinds_of_int = [torch.tensor(4), torch.tensor([0, 5])[-1], torch.tensor([3]), np.int64(-7), np.array(6), True, 2 ** 40 + 1,
                    torch.zeros(3, dtype=torch.int32), torch.tensor(4.0), None, 4.0, "4", object()]
    for name in ("kvattn_cache_write", "kvattn_decode", "kvattn_append_decode", "kvattn_paged_cache_write",
                 "kvattn_paged_decode", "kvattn_paged_decode_tokens", "kvattn_paged_reserve", "kvattn_paged_store",
                 "kvattn_paged_load", "kvattn_verify_drafts"):
        kinds = kvattn.SIGNATURES[name][1]
        for i, k in enumerate(kinds):
            if k is kvattn._vp:
                continue
            for x in kinds_of_int:
                # Every other integer fits, and the pointers are missing: refused, by the sizes or for a pointer.
                args = [None if t is kvattn._vp else 64 for t in kinds]
                args[i] = x
                try:
                    want = getattr(kvattn.lib(), name)(*args)
                except ctypes.ArgumentError:
                    with pytest.raises(ctypes.ArgumentError):
                        getattr(kvattn._call, name)(*args)
                    continue
                assert want != kvattn.OK and getattr(kvattn._call, name)(*args) == want, (name, i, x)


@pytest.mark.parametrize("extension", [True, False])
def test_counts_of_wrappers_are_values(monkeypatch, extension):
    """The statuses tell whether a count arrived: -1 is refused as a size before the missing pointer is."""
    import torch
    kvattn = _calls(monkeypatch, extension)
    x = torch.zeros(64, dtype=torch.int32)
    cache = kvattn.PagedCache(x, x, 1, 64, 1, x)
    for n, status in ((torch.tensor([0, -1])[-1], kvattn.ERR_SHAPE), (torch.tensor(2), kvattn.ERR_NULL_POINTER)):
        for call in (lambda: kvattn.decode(None, None, None, n, 1, 64, 64, kv_dtype="bf16", stream=0),
                     lambda: kvattn.append_decode(None, None, None, 1, n, 64, 64, kv_dtype="bf16", stream=0),
                     lambda: kvattn.kv_cache_write(None, None, 1, 1, 64, n, kv_dtype="bf16", stream=0),
                     lambda: kvattn.paged_decode(None, None, cache, n, 1, 64, kv_dtype="bf16", stream=0),
                     lambda: kvattn.paged_decode_tokens(None, x, cache, x, x, 1, n, 1, 64, kv_dtype="int4", max_new=1, stream=0),
                     lambda: kvattn.paged_store(cache, None, x, n, 1, 64, kv_dtype="bf16", stream=0),
                     lambda: kvattn.verify_drafts(x, x, None, x, x, x, 1, n, 8, stream=0)):
            with pytest.raises(kvattn.KvAttnError) as e:
                call()
            assert e.value.status == status


def test_integers_by_bit():
    import torch
    from cuda_gpt2_inference_amd._pycall import Call
    got = []

    def seen(*words):
        got[:] = words
        return 0
    fn = ctypes.CFUNCTYPE(ctypes.c_int, *[_W] * 24)(seen)
    call = Call(ctypes.cast(fn, ctypes.c_void_p).value, 24, 0b101 | 1 << 23)
    x = torch.zeros(2)
    assert call(np.int64(-7), x, torch.tensor(9), *[x] * 20, 2 ** 64 + 3) == 0
    assert got == [-7, x.data_ptr(), 9] + [x.data_ptr()] * 20 + [3]
    for i in (0, 2, 23):
        args = [1] * 24
        args[i] = x
        with pytest.raises(ctypes.ArgumentError, match=f"argument {i + 1}:"):
            call(*args)
