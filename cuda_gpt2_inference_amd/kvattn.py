"""ctypes binding of libkvattn.so (the C ABI declared in include/kvattn.h).

Two layers:

* ``lib()`` returns the loaded library with every entry point's argtypes/restype set;
  arguments are raw device pointers (ints) and sizes, exactly the C ABI.
* The functions named after the reference's host entry points
  (``kv_cache_write``, ``attention_forward_kv_small``, ``attention_forward_kv_large``,
  ``attention_kv_split``, ``attention_kv_merge``) and ``decode`` accept torch tensors
  (or raw pointers), pass ``torch.cuda.current_stream()`` unless a stream is given, and
  raise ``KvAttnError`` on a non-zero status -- the reference's ``cudaCheck`` prints and
  exits (Inference_gpt2/common.h:123-130); a Python caller gets an exception instead.

There is no fallback: if the shared library is missing, importing the binding works
but the first call raises ``KvAttnError`` telling the caller to build it.
"""
from __future__ import annotations

import ctypes
import os
from typing import Optional

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libkvattn.so")

# kvattn_status
OK = 0
ERR_NULL_POINTER = 1
ERR_MISALIGNED = 2
ERR_HEAD_DIM = 3
ERR_SHAPE = 4
ERR_DTYPE = 5
ERR_STRATEGY = 6
ERR_WORKSPACE = 7
ERR_SPLIT = 8
ERR_COOP_TOO_LARGE = 9
ERR_LDS = 10
ERR_CAPTURE = 11
ERR_LENGTH = 12
ERR_HIP = 13
ERR_GRID_TOO_LARGE = 14
ERR_MERGE_TIMEOUT = 15

# kvattn_dtype
KV_F32 = 0
KV_BF16 = 1
KV_INT8 = 2
KV_FP8_E4M3 = 3
KV_INT4 = 4
KV_FP4_E2M1 = 5
KV_DTYPES = {"f32": KV_F32, "bf16": KV_BF16, "int8": KV_INT8, "fp8": KV_FP8_E4M3, "int4": KV_INT4,
             "fp4": KV_FP4_E2M1}

# kvattn_strategy
AUTO = 0
FUSED_SINGLE = 1
SPLIT_MERGE = 2
SINGLE_LAUNCH_COOP = 3
SINGLE_LAUNCH_GRAPH = 4
SPLIT_LASTBLOCK = 5
SPLIT_DESIGNATED = 6
STRATEGIES = {
    "auto": AUTO,
    "fused_single": FUSED_SINGLE,
    "split_merge": SPLIT_MERGE,
    "coop": SINGLE_LAUNCH_COOP,
    "graph": SINGLE_LAUNCH_GRAPH,
    "lastblock": SPLIT_LASTBLOCK,
    "designated": SPLIT_DESIGNATED,
}

HEAD_DIM = 64

_vp = ctypes.c_void_p
_i = ctypes.c_int
_ll = ctypes.c_longlong
_sz = ctypes.c_size_t

# name -> (restype, argtypes); mirrors include/kvattn.h one to one.
SIGNATURES = {
    "kvattn_strerror": (ctypes.c_char_p, [_i]),
    "kvattn_last_hip_error": (_i, []),
    "kvattn_cur_len_symbol": (_i, [ctypes.POINTER(_vp)]),
    "kvattn_set_cur_len": (_i, [_i]),
    "kvattn_set_cur_len_async": (_i, [_vp, _i, _vp]),
    "kvattn_cache_write": (_i, [_vp, _vp, _vp, _i, _i, _i, _i, _vp, _i, _i, _vp]),
    "kvattn_append": (_i, [_vp, _vp, _vp, _i, _i, _i, _i, _vp, _i, _vp]),
    "kvattn_forward_small": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _i, _i, _vp]),
    "kvattn_forward_large": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _i, _vp, _vp, _vp, _i, _i, _vp]),
    "kvattn_split": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _i, _i, _i, _vp]),
    "kvattn_merge": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp]),
    "kvattn_workspace_bytes": (_sz, [_i, _i, _i, _i, _i]),
    "kvattn_workspace_init": (_i, [_vp, _sz, _vp]),
    "kvattn_workspace_status": (_i, [_vp, _sz, _i, _vp, ctypes.POINTER(_i)]),
    "kvattn_set_merge_poll_limit": (_i, [_i]),
    "kvattn_scratch_status": (_i, [_i, _vp, ctypes.POINTER(_i)]),
    "kvattn_call_identity": (_i, [_vp, _vp]),
    "kvattn_set_xcd_layout_offset": (_i, [_i]),
    "kvattn_plan": (_i, [_i, _i, _i, _i, _i, _i, _i, _i, ctypes.POINTER(_i), ctypes.POINTER(_i),
                         ctypes.POINTER(_i)]),
    "kvattn_decode": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _i, _i, _vp, _sz, _i, _i, _i, _vp]),
    "kvattn_append_decode": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _i, _i, _vp, _sz, _i, _i, _i, _vp]),
    "kvattn_decode_static": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _i, _i, _i, _i, _i, _vp]),
    "kvattn_gemv": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp]),
    "kvattn_gemv_ex": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _vp]),
    "kvattn_gemv_qkv_append": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _vp, _i, _vp, _i, _i, _i, _vp,
                                    _sz, _vp]),
    "kvattn_gemv_qkv_append_workspace_bytes": (_sz, [_i, _i]),
    "kvattn_paged_cache_write": (_i, [_vp, _vp, _vp, _i, _i, _i, _vp, _i, _i, _i, _vp, _i, _i, _vp]),
    "kvattn_paged_decode": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _vp, _i, _i, _vp, _sz, _i, _i,
                                 _i, _i, _vp]),
    "kvattn_paged_decode_tokens": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp, _vp, _i, _i, _i, _i, _i, _vp, _sz,
                                        _i, _i, _vp]),
    "kvattn_paged_pool_bytes": (_sz, [_i]),
    "kvattn_paged_pool_init": (_i, [_vp, _i, _vp]),
    "kvattn_paged_reserve": (_i, [_vp, _i, _i, _i, _vp, _vp, _vp, _vp, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp]),
    "kvattn_paged_store": (_i, [_vp, _vp, _i, _i, _vp, _vp, _i, _i, _i, _i, _vp]),
    "kvattn_paged_load": (_i, [_vp, _vp, _vp, _i, _i, _vp, _i, _i, _i, _i, _vp]),
    "kvattn_verify_workspace_bytes": (_sz, [_i, _i]),
    "kvattn_verify_drafts": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _ll, _i, _vp, _sz, _vp]),
    "kvattn_tree_masks": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp]),
    "kvattn_paged_decode_tree": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _vp,
                                      _sz, _i, _i, _vp]),
    "kvattn_paged_keep": (_i, [_vp, _vp, _i, _i, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp]),
    "kvattn_verify_tree": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _ll, _i, _vp, _sz,
                                _vp]),
    "kvattn_logits_workspace_bytes": (_sz, []),
    "kvattn_process_logits": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _ll, _ll, _i, _i, _i, _vp]),
    "kvattn_w4_bytes": (_sz, [_i, _i, _i]),
    "kvattn_w4_pack": (_i, [_vp, _vp, _vp, _i, _i, _i, _i, _vp]),
    "kvattn_w4_quantize": (_i, [_vp, _vp, _i, _i, _i, _i, _i, _vp]),
    "kvattn_gemv_w4": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _vp]),
}


class KvAttnError(RuntimeError):
    def __init__(self, status: int, where: str):
        self.status = status
        text = strerror(status) if _LIB is not None else "library not loaded"
        hip = ""
        if status == ERR_HIP and _LIB is not None:
            hip = f" (hipError {_LIB.kvattn_last_hip_error()})"
        super().__init__(f"{where}: kvattn status {status}: {text}{hip}")


_LIB: Optional[ctypes.CDLL] = None


def lib() -> ctypes.CDLL:
    """Load libkvattn.so once; raise if it has not been built."""
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise KvAttnError(-1, f"{LIB_PATH} is missing; build it with __graft_entry__.build() "
                                  "or `make -C cuda_gpt2_inference_amd/csrc`")
        handle = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _LIB = handle
    return _LIB


def strerror(status: int) -> str:
    return lib().kvattn_strerror(status).decode()


def _check(status: int, where: str) -> None:
    if status != OK:
        raise KvAttnError(status, where)


def _ptr(x) -> Optional[int]:
    """Device address of a tensor, an int address, or None."""
    if x is None:
        return None
    if isinstance(x, int):
        return x
    return x.data_ptr()


class _Calls:
    """The entry points that return a status, bound at their first use: each takes tensors, addresses and None as
    they are where it has a pointer, and an integer's value where it has an integer (_pycall.Call; without it
    ctypes, and _ptr for every pointer).  What is no integer there is a ctypes.ArgumentError."""

    def __getattr__(self, name):
        fn = getattr(lib(), name)
        kinds = SIGNATURES[name][1]
        try:
            from ._pycall import Call
        except ImportError:
            def call(*args):
                if len(args) != len(kinds):
                    raise TypeError(f"{len(kinds)} positional arguments expected, {len(args)} given")
                return fn(*[_ptr(x) if k is _vp else x for k, x in zip(kinds, args)])
        else:
            call = Call(ctypes.cast(fn, _vp).value, len(kinds), sum(1 << i for i, k in enumerate(kinds) if k is not _vp))
        setattr(self, name, call)
        return call


_call = _Calls()


# The handle of torch's current stream on the current device.  torch.cuda.current_stream() builds
# a Stream object for it, 2.8 us of an eager call's 8.3 us; the handle alone takes 0.1 us.
_current_stream = None


def _find_current_stream():
    import torch
    raw, device = getattr(torch._C, "_cuda_getCurrentRawStream", None), torch.cuda.current_device
    if raw is None:
        return lambda: torch.cuda.current_stream().cuda_stream
    return lambda: raw(device())


def _stream(stream) -> Optional[int]:
    if stream is None:
        global _current_stream
        if _current_stream is None:
            _current_stream = _find_current_stream()
        return _current_stream()
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def kv_dtype_code(kv_dtype) -> int:
    if isinstance(kv_dtype, str):
        return KV_DTYPES[kv_dtype]
    return int(kv_dtype)


def strategy_code(strategy) -> int:
    if isinstance(strategy, str):
        return STRATEGIES[strategy]
    return int(strategy)


def cur_len_symbol() -> int:
    """Device address of the library's own device-resident length."""
    p = _vp()
    _check(lib().kvattn_cur_len_symbol(ctypes.byref(p)), "kvattn_cur_len_symbol")
    return int(p.value)


def set_cur_len(cur_len: int) -> None:
    _check(lib().kvattn_set_cur_len(int(cur_len)), "kvattn_set_cur_len")


def set_cur_len_async(cur_len: int, d_cur_len=None, stream=None) -> None:
    """Stream-ordered write of the device length (no host synchronisation)."""
    _check(lib().kvattn_set_cur_len_async(_ptr(d_cur_len), int(cur_len), _stream(stream)),
           "kvattn_set_cur_len_async")


def kv_cache_write(kv_cache, qkv, B, NH, hs, maxT, *, kv_dtype, kv_scale=None, cur_len=None,
                   lens_per_seq=False, stream=None) -> None:
    """Append the current token's K/V (reference kv_cache_write_kernel[_w8])."""
    _check(_call.kvattn_cache_write(kv_cache, kv_scale, qkv, B, NH, hs, maxT, cur_len,
                                    int(bool(lens_per_seq)), kv_dtype_code(kv_dtype),
                                    _stream(stream)), "kvattn_cache_write")


def attention_forward_kv_small(out, qkv, kv_cache, B, NH, hs, maxT, *, kv_dtype, kv_scale=None,
                               cur_len=None, lens_per_seq=False, stream=None) -> None:
    """fused_single (reference attention_forward_kv_small[_w8])."""
    _check(lib().kvattn_forward_small(_ptr(out), _ptr(qkv), _ptr(kv_cache), _ptr(kv_scale), B, NH, hs, maxT,
                                      _ptr(cur_len), int(bool(lens_per_seq)), kv_dtype_code(kv_dtype),
                                      _stream(stream)), "kvattn_forward_small")


def attention_forward_kv_large(out, qkv, kv_cache, B, NH, hs, maxT, part_out, part_lse, part_max, S, *,
                               kv_dtype, kv_scale=None, cur_len=None, lens_per_seq=False,
                               stream=None) -> None:
    """Split + merge or cooperative (reference attention_forward_kv_large[_w8])."""
    _check(lib().kvattn_forward_large(_ptr(out), _ptr(qkv), _ptr(kv_cache), _ptr(kv_scale), B, NH, hs, maxT,
                                      _ptr(cur_len), int(bool(lens_per_seq)), _ptr(part_out), _ptr(part_lse),
                                      _ptr(part_max), S, kv_dtype_code(kv_dtype), _stream(stream)),
           "kvattn_forward_large")


def attention_kv_split(part_out, part_lse, part_max, qkv, kv_cache, B, NH, hs, maxT, S, *, kv_dtype,
                       kv_scale=None, cur_len=None, lens_per_seq=False, stream=None) -> None:
    """Split phase (reference attention_kv_split_kernel[_w8])."""
    _check(lib().kvattn_split(_ptr(part_out), _ptr(part_lse), _ptr(part_max), _ptr(qkv), _ptr(kv_cache),
                              _ptr(kv_scale), B, NH, hs, maxT, _ptr(cur_len), int(bool(lens_per_seq)), S,
                              kv_dtype_code(kv_dtype), _stream(stream)), "kvattn_split")


def attention_kv_merge(out, part_out, part_lse, part_max, B, NH, hs, S, *, kv_dtype, stream=None) -> None:
    """Merge phase (reference attention_kv_merge_kernel[_w8])."""
    _check(lib().kvattn_merge(_ptr(out), _ptr(part_out), _ptr(part_lse), _ptr(part_max), B, NH, hs, S,
                              kv_dtype_code(kv_dtype), _stream(stream)), "kvattn_merge")


def workspace_bytes(B, NH, hs, maxT, S=0) -> int:
    return int(lib().kvattn_workspace_bytes(B, NH, hs, maxT, S))


def workspace_init(workspace, nbytes, stream=None) -> None:
    _check(lib().kvattn_workspace_init(_ptr(workspace), nbytes, _stream(stream)), "kvattn_workspace_init")


def workspace_status(workspace, nbytes, clear=False, stream=None) -> int:
    """Merges that stopped waiting since the workspace was initialised or last cleared
    (kvattn_workspace_status; synchronises the stream): designated mergers that computed
    their producers' segments themselves, cooperative mergers that wrote NaN.  Returns the
    count; it is not an error to find one here."""
    n = _i()
    st = lib().kvattn_workspace_status(_ptr(workspace), int(nbytes), int(bool(clear)), _stream(stream),
                                       ctypes.byref(n))
    if st not in (OK, ERR_MERGE_TIMEOUT):
        _check(st, "kvattn_workspace_status")
    return n.value


def scratch_status(clear=False, stream=None) -> int:
    """Merges that stopped waiting in the library's static scratch array on the current device
    (kvattn_scratch_status; the workspace of decode_static and of forward_large's single
    launch; synchronises the stream).  Returns the count."""
    n = _i()
    st = lib().kvattn_scratch_status(int(bool(clear)), _stream(stream), ctypes.byref(n))
    if st not in (OK, ERR_MERGE_TIMEOUT):
        _check(st, "kvattn_scratch_status")
    return n.value


def call_identity(out, stream=None) -> None:
    """Enqueue one dispatch that writes {dispatch id, queue address, tag} into out (3 int64
    words on the device): the identity a tagged partial word of that stream carries."""
    _check(lib().kvattn_call_identity(_ptr(out), _stream(stream)), "kvattn_call_identity")


def set_xcd_layout_offset(rot: int) -> int:
    """Test setting: designated producers `rot` XCDs away from their merger (0: the layout in
    use).  Returns the previous setting."""
    return int(lib().kvattn_set_xcd_layout_offset(int(rot)))


def set_merge_poll_limit(polls: int) -> int:
    """Bound on a merger's polls for later launches (0: stop waiting at once, a
    fault-injection setting; < 0: the default, 2^16).  Returns the previous bound."""
    return int(lib().kvattn_set_merge_poll_limit(int(polls)))


def plan(B, NH, hs, maxT, *, kv_dtype, len_hint=-1, S=0, strategy="auto"):
    """(strategy code, segment slots per (b,h) its workspace must hold, rows per segment) of kvattn_decode."""
    st, seg, rows = _i(), _i(), _i()
    _check(lib().kvattn_plan(B, NH, hs, maxT, int(len_hint), int(S), strategy_code(strategy),
                             kv_dtype_code(kv_dtype), ctypes.byref(st), ctypes.byref(seg), ctypes.byref(rows)),
           "kvattn_plan")
    return st.value, seg.value, rows.value


STRATEGY_NAMES = {v: k for k, v in STRATEGIES.items()}


def decode(out, qkv, kv_cache, B, NH, hs, maxT, *, kv_dtype, kv_scale=None, cur_len=None,
           lens_per_seq=False, len_hint=-1, workspace=None, workspace_nbytes=0, S=0, strategy="auto",
           stream=None) -> None:
    """One decode-attention call with an explicit strategy (kvattn_decode)."""
    _check(_call.kvattn_decode(out, qkv, kv_cache, kv_scale, B, NH, hs, maxT,
                               cur_len, int(bool(lens_per_seq)), int(len_hint), workspace,
                               int(workspace_nbytes), int(S), strategy_code(strategy),
                               kv_dtype_code(kv_dtype), _stream(stream)), "kvattn_decode")


def decode_static(out, qkv, kv_cache, B, NH, hs, maxT, *, kv_dtype, kv_scale=None, cur_len=None,
                  lens_per_seq=False, len_hint=-1, S=0, strategy="auto", stream=None) -> None:
    """decode with the library's static device scratch as workspace (kvattn_decode_static):
    allocates nothing; calls that overlap in time on one GPU race."""
    _check(lib().kvattn_decode_static(_ptr(out), _ptr(qkv), _ptr(kv_cache), _ptr(kv_scale), B, NH, hs, maxT,
                                      _ptr(cur_len), int(bool(lens_per_seq)), int(len_hint), int(S),
                                      strategy_code(strategy), kv_dtype_code(kv_dtype), _stream(stream)),
           "kvattn_decode_static")


def append_decode(out, qkv, kv_cache, B, NH, hs, maxT, *, kv_dtype, kv_scale=None, cur_len=None,
                  lens_per_seq=False, len_hint=-1, workspace=None, workspace_nbytes=0, S=0, strategy="auto",
                  stream=None) -> None:
    """kv_cache_write + decode in one launch (kvattn_append_decode)."""
    _check(_call.kvattn_append_decode(out, qkv, kv_cache, kv_scale, B, NH, hs, maxT,
                                      cur_len, int(bool(lens_per_seq)), int(len_hint), workspace,
                                      int(workspace_nbytes), int(S), strategy_code(strategy),
                                      kv_dtype_code(kv_dtype), _stream(stream)), "kvattn_append_decode")


def gemv(out, W, x, B, M, K, *, w_dtype, w_scale=None, bias=None, pre_gelu=None, gelu=False, out_dtype=None,
         stream=None) -> None:
    """Decode-step fully connected layer out = [GELU](W x [* w_scale] + bias) (kvattn_gemv;
    kvattn_gemv_ex when out_dtype, "f32" or "bf16", is given)."""
    if out_dtype is None:
        _check(lib().kvattn_gemv(_ptr(out), _ptr(pre_gelu), _ptr(W), _ptr(w_scale), _ptr(x), _ptr(bias), B, M, K,
                                 kv_dtype_code(w_dtype), int(bool(gelu)), _stream(stream)), "kvattn_gemv")
        return
    _check(lib().kvattn_gemv_ex(_ptr(out), _ptr(pre_gelu), _ptr(W), _ptr(w_scale), _ptr(x), _ptr(bias), B, M, K,
                                kv_dtype_code(w_dtype), kv_dtype_code(out_dtype), int(bool(gelu)),
                                _stream(stream)), "kvattn_gemv_ex")


def gemv_qkv_append(qkv, W, x, B, NH, hs, K, kv_cache, maxT, *, w_dtype, kv_dtype=None, w_scale=None, bias=None,
                    kv_scale=None, cur_len=None, lens_per_seq=False, workspace=None, workspace_nbytes=0,
                    stream=None) -> None:
    """QKV projection with the KV append in its epilogue (kvattn_gemv_qkv_append).  kv_dtype
    defaults to the activation type (f32 for f32 weights, else bf16); 8-bit caches need
    kv_scale and a workspace of gemv_qkv_append_workspace_bytes(B, NH), zeroed once."""
    if kv_dtype is None:
        kv_dtype = "f32" if kv_dtype_code(w_dtype) == KV_F32 else "bf16"
    _check(lib().kvattn_gemv_qkv_append(_ptr(qkv), _ptr(W), _ptr(w_scale), _ptr(x), _ptr(bias), B, NH, hs, K,
                                        _ptr(kv_cache), _ptr(kv_scale), maxT, _ptr(cur_len),
                                        int(bool(lens_per_seq)), kv_dtype_code(w_dtype), kv_dtype_code(kv_dtype),
                                        _ptr(workspace), int(workspace_nbytes), _stream(stream)),
           "kvattn_gemv_qkv_append")


def gemv_qkv_append_workspace_bytes(B: int, NH: int) -> int:
    """Workspace bytes gemv_qkv_append needs for an 8-bit cache."""
    return int(lib().kvattn_gemv_qkv_append_workspace_bytes(B, NH))


class PagedCache:
    """A paged KV cache: a page pool [num_pages][2][NH][page_rows][hs] (hs / 2 bytes a row for 4-bit
    caches; + row scales for 8-bit and 4-bit caches) and a block table [B][max_pages] of page ids
    (device tensors)."""

    def __init__(self, pages, block_table, max_pages, page_rows, num_pages, page_scales=None):
        self.pages, self.block_table, self.page_scales = pages, block_table, page_scales
        self.max_pages, self.page_rows, self.num_pages = int(max_pages), int(page_rows), int(num_pages)

    @property
    def maxT(self) -> int:
        return self.max_pages * self.page_rows

    def _args(self):
        return (self.pages, self.page_scales, self.block_table, self.max_pages, self.page_rows,
                self.num_pages)


def paged_cache_write(cache: PagedCache, qkv, B, NH, hs, *, kv_dtype, cur_len=None, lens_per_seq=False,
                      stream=None) -> None:
    """kv_cache_write into a paged cache (kvattn_paged_cache_write)."""
    _check(_call.kvattn_paged_cache_write(*cache._args(), qkv, B, NH, hs, cur_len,
                                          int(bool(lens_per_seq)), kv_dtype_code(kv_dtype), _stream(stream)),
           "kvattn_paged_cache_write")


def paged_decode(out, qkv, cache: PagedCache, B, NH, hs, *, kv_dtype, cur_len=None, lens_per_seq=False,
                 len_hint=-1, workspace=None, workspace_nbytes=0, S=0, strategy="auto", append=False,
                 stream=None) -> None:
    """decode / append_decode on a paged cache (kvattn_paged_decode)."""
    p = cache._args()
    _check(_call.kvattn_paged_decode(out, qkv, p[0], p[1], p[2], p[3], p[4], p[5], B, NH, hs,
                                     cur_len, int(bool(lens_per_seq)), int(len_hint), workspace,
                                     int(workspace_nbytes), int(S), strategy_code(strategy),
                                     kv_dtype_code(kv_dtype), int(bool(append)), _stream(stream)),
           "kvattn_paged_decode")


def paged_decode_tokens(out, qkv, cache: PagedCache, token_start, lens, B, num_tokens, NH, hs, *, kv_dtype, max_new,
                        workspace=None, workspace_nbytes=0, S=0, stream=None) -> None:
    """Attention of several new tokens of every sequence over a paged 4-bit cache that holds their rows
    (kvattn_paged_decode_tokens); the workspace is that of num_tokens sequences."""
    _check(_call.kvattn_paged_decode_tokens(out, qkv, cache.pages, cache.page_scales, cache.block_table,
                                            cache.max_pages, cache.page_rows, cache.num_pages, token_start, lens, B,
                                            num_tokens, int(max_new), NH, hs, workspace, int(workspace_nbytes),
                                            int(S), kv_dtype_code(kv_dtype),
                                            _stream(stream)), "kvattn_paged_decode_tokens")


def paged_pool(num_pages, device="cuda", stream=None):
    """A pool of free pages for paged_reserve: int32 [4 + num_pages], every page free."""
    import torch
    nbytes = int(lib().kvattn_paged_pool_bytes(int(num_pages)))
    if nbytes == 0:
        raise KvAttnError(ERR_SHAPE, "kvattn_paged_pool_bytes")
    pool = torch.empty(nbytes // 4, dtype=torch.int32, device=device)
    with torch.cuda.device(pool.device):
        _check(lib().kvattn_paged_pool_init(_ptr(pool), int(num_pages), _stream(stream)), "kvattn_paged_pool_init")
    return pool


def paged_reserve(cache: PagedCache, pool, held, kept, fresh, B, *, lens, token_start, slot_map, max_tokens,
                  held_out=None, positions=None, pool_next=None, stream=None) -> None:
    """Pages, token offsets, slot map and positions of a step from what every request holds, keeps and
    adds (kvattn_paged_reserve).  held_out None: held is updated in place."""
    _check(_call.kvattn_paged_reserve(cache.block_table, cache.max_pages, cache.page_rows, cache.num_pages,
                                      pool, held, kept, fresh, B, int(max_tokens),
                                      held if held_out is None else held_out, lens, token_start, slot_map,
                                      positions, pool_next, _stream(stream)),
           "kvattn_paged_reserve")


def paged_store(cache: PagedCache, qkv, slot_map, num_tokens, NH, hs, *, kv_dtype, stream=None) -> None:
    """K and V of a batch of tokens into the pool by slot (kvattn_paged_store)."""
    _check(_call.kvattn_paged_store(cache.pages, cache.page_scales, cache.page_rows, cache.num_pages,
                                    slot_map, qkv, num_tokens, NH, hs, kv_dtype_code(kv_dtype),
                                    _stream(stream)), "kvattn_paged_store")


def paged_load(kv, cache: PagedCache, slot_map, num_tokens, NH, hs, *, kv_dtype, stream=None) -> None:
    """Rows of the pool by slot into kv [num_tokens][2][NH][hs] (kvattn_paged_load)."""
    _check(_call.kvattn_paged_load(kv, cache.pages, cache.page_scales, cache.page_rows,
                                   cache.num_pages, slot_map, num_tokens, NH, hs, kv_dtype_code(kv_dtype),
                                   _stream(stream)), "kvattn_paged_load")


def verify_workspace_bytes(B, V) -> int:
    """Workspace bytes of verify_drafts, to be zeroed once with workspace_init."""
    return int(lib().kvattn_verify_workspace_bytes(B, V))


def verify_drafts(tokens, counts, target_probs, draft_tokens, uniform, token_start, B, num_tokens, V, *,
                  draft_probs=None, row_stride=None, dtype="f32", workspace=None, workspace_nbytes=0,
                  stream=None) -> None:
    """Accepts drafted tokens against the target's probabilities and draws the next one
    (kvattn_verify_drafts).  draft_probs None: drafts without probabilities."""
    _check(_call.kvattn_verify_drafts(tokens, counts, target_probs, draft_probs,
                                      draft_tokens, uniform, token_start, B, num_tokens, V,
                                      V if row_stride is None else int(row_stride), kv_dtype_code(dtype),
                                      workspace, int(workspace_nbytes), _stream(stream)), "kvattn_verify_drafts")


def tree_masks(masks, parents, token_start, B, num_tokens, *, positions=None, lens=None, mask_words=1, stream=None) -> None:
    """Masks (and positions) of trees of drafted tokens from every token's parent (kvattn_tree_masks)."""
    _check(_call.kvattn_tree_masks(masks, positions, parents, token_start, lens, B, num_tokens, int(mask_words),
                                   _stream(stream)), "kvattn_tree_masks")


def paged_decode_tree(out, qkv, cache: PagedCache, token_start, lens, masks, B, num_tokens, NH, hs, *, kv_dtype, max_new,
                      mask_words=1, workspace=None, workspace_nbytes=0, S=0, stream=None) -> None:
    """Attention of trees of drafted tokens over a paged cache that holds their rows (kvattn_paged_decode_tree); the
    workspace is that of num_tokens sequences."""
    _check(_call.kvattn_paged_decode_tree(out, qkv, cache.pages, cache.page_scales, cache.block_table, cache.max_pages,
                                          cache.page_rows, cache.num_pages, token_start, lens, masks, int(mask_words), B,
                                          num_tokens, int(max_new), NH, hs, workspace, int(workspace_nbytes), int(S),
                                          kv_dtype_code(kv_dtype), _stream(stream)), "kvattn_paged_decode_tree")


def paged_keep(cache: PagedCache, slot_map, path, token_start, B, num_tokens, NH, hs, *, kv_dtype, stream=None) -> None:
    """K and V rows of the accepted paths to where the next step needs them (kvattn_paged_keep)."""
    _check(_call.kvattn_paged_keep(cache.pages, cache.page_scales, cache.page_rows, cache.num_pages, slot_map, path,
                                   token_start, B, num_tokens, NH, hs, kv_dtype_code(kv_dtype), _stream(stream)),
           "kvattn_paged_keep")


def verify_tree(tokens, path, counts, target_probs, tree_tokens, parents, uniform, draw, token_start, B, num_tokens, V, *,
                lens=None, kept=None, row_stride=None, dtype="f32", workspace=None, workspace_nbytes=0,
                stream=None) -> None:
    """Accepts a path of a tree of drafted tokens against the target's probabilities and draws the next token
    (kvattn_verify_tree); the workspace is verify_drafts'."""
    _check(_call.kvattn_verify_tree(tokens, path, counts, kept, target_probs, tree_tokens, parents, uniform, draw,
                                    token_start, lens, B, num_tokens, V, V if row_stride is None else int(row_stride),
                                    kv_dtype_code(dtype), workspace, int(workspace_nbytes), _stream(stream)),
           "kvattn_verify_tree")


class _LogitRules(ctypes.Structure):
    """kvattn_logit_rules."""
    _fields_ = [(name, _vp) for name in (
        "history", "history_len", "prompt_len", "tokens", "masks", "repetition", "frequency", "presence", "bias_start",
        "bias_ids", "bias", "allowed", "allowed_of", "temperature")] + [
        (name, _i) for name in ("max_history", "mask_words", "num_bias", "max_bias", "num_allowed", "allowed_stride")] + [
        ("workspace", _vp), ("workspace_bytes", _sz)]


class LogitRules:
    """Rules on logits for process_logits: the fields of kvattn_logit_rules by name, device tensors and integers.  Made
    once; the tensors are kept, and may be written between calls.  Without a workspace of the caller's, rules with tensors
    bring their own, so calls with one LogitRules must be ordered."""

    def __init__(self, **rules):
        self._struct = _LogitRules()
        like = next((x for x in rules.values() if hasattr(x, "device")), None)
        if "workspace" not in rules and like is not None and like.is_cuda:
            import torch
            nbytes = int(lib().kvattn_logits_workspace_bytes())
            rules = dict(rules, workspace=torch.zeros(nbytes, dtype=torch.uint8, device=like.device), workspace_bytes=nbytes)
        names = dict(_LogitRules._fields_)
        for name, x in rules.items():
            if name not in names:
                raise TypeError(f"LogitRules: no rule {name!r}")
            setattr(self._struct, name, _ptr(x) if names[name] is _vp else int(x))
        self._tensors = rules
        self.address = ctypes.addressof(self._struct)


def process_logits(out, logits, rules: Optional[LogitRules], token_start, B, rows, V, *, row_stride=None, out_stride=None,
                   dtype="f32", out_dtype=None, probs=True, stream=None) -> None:
    """Penalties, biases and grammar masks on rows of logits, as probabilities (or, probs False, as logits)
    (kvattn_process_logits).  out_dtype None: dtype."""
    _check(_call.kvattn_process_logits(out, logits, None if rules is None else rules.address, token_start, B, rows, V,
                                       V if row_stride is None else int(row_stride),
                                       V if out_stride is None else int(out_stride), kv_dtype_code(dtype),
                                       kv_dtype_code(dtype if out_dtype is None else out_dtype), int(bool(probs)),
                                       _stream(stream)), "kvattn_process_logits")


def w4_bytes(M, K, group) -> int:
    """Bytes of an M x K matrix of 4-bit weights as gemv_w4 reads it."""
    return int(lib().kvattn_w4_bytes(M, K, group))


def _w4_buffer(M, K, group, like):
    import torch
    nbytes = w4_bytes(M, K, group)
    if nbytes == 0:
        raise KvAttnError(ERR_SHAPE, "kvattn_w4_bytes")
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device)


def w4_pack(codes, scales, M, K, group, *, w_dtype, out=None, stream=None):
    """4-bit codes [M][K/2] and bf16 scales [M][K/group] laid out for gemv_w4 (kvattn_w4_pack)."""
    out = _w4_buffer(M, K, group, codes) if out is None else out
    _check(_call.kvattn_w4_pack(out, codes, scales, M, K, int(group), kv_dtype_code(w_dtype), _stream(stream)), "kvattn_w4_pack")
    return out


def w4_quantize(W, M, K, group, *, w_dtype, src_dtype="bf16", out=None, stream=None):
    """W [M][K] coded in 4 bits and laid out for gemv_w4 (kvattn_w4_quantize)."""
    out = _w4_buffer(M, K, group, W) if out is None else out
    _check(_call.kvattn_w4_quantize(out, W, M, K, int(group), kv_dtype_code(src_dtype), kv_dtype_code(w_dtype),
                                    _stream(stream)), "kvattn_w4_quantize")
    return out


def gemv_w4(out, w4, x, B, M, K, *, group, w_dtype, bias=None, pre_gelu=None, gelu=False, out_dtype="bf16", stream=None) -> None:
    """Fully connected layer on 4-bit weights with a scale for every group (kvattn_gemv_w4)."""
    _check(_call.kvattn_gemv_w4(out, pre_gelu, w4, x, bias, B, M, K, int(group), kv_dtype_code(w_dtype),
                                kv_dtype_code(out_dtype), int(bool(gelu)), _stream(stream)), "kvattn_gemv_w4")


class Workspace:
    """Device workspace for ``decode``: allocated with torch, counters zeroed once."""

    def __init__(self, B, NH, maxT, S=0, device="cuda"):
        import torch
        self.nbytes = workspace_bytes(B, NH, HEAD_DIM, maxT, S)
        if self.nbytes == 0:
            raise KvAttnError(ERR_SHAPE, "kvattn_workspace_bytes")
        self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=device)
        workspace_init(self.buf, self.nbytes)

    def kwargs(self):
        return {"workspace": self.buf, "workspace_nbytes": self.nbytes}

    def status(self, clear=False, stream=None) -> int:
        """Designated merges on this workspace that stopped waiting (see workspace_status)."""
        return workspace_status(self.buf, self.nbytes, clear=clear, stream=stream)
