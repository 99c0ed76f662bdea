"""The operators of a speculative serving step over a paged 4-bit KV cache, as timed cases.

Four kinds of case:

  attn    decode attention over a 4-bit cache (INT4 or FP4 E2M1 codes, one float scale per row of
          64 channels): one token a sequence over a contiguous cache (``decode``) or a paged one
          (``paged_decode``), or several new tokens a sequence, each attending the positions up
          to its own (``paged_decode_tokens``)
  tables  block tables, token offsets, slot map and positions of a step, from what every request
          holds, keeps and adds (``paged_reserve``)
  rows    K and V of a step's tokens into the pool by slot map, and back out of it as prefill
          attention reads them (``paged_store``, ``paged_load``)
  verify  drafted tokens against the target's probabilities (``verify_drafts``)

With ``own`` the calls go to ``cuda_gpt2_inference_amd.kvattn``; without, they are computed with
elementary torch operations in 32 bits (the draws of ``verify`` in 64).
"""
import math

import torch

own = False

HD = 64
VOCAB, VOCAB_ROW = 50257, 50304      # GPT-2's tokens, and the padded row of its logits
LIMIT = {"int4": 7.0, "fp4": 6.0, "int8": 127.0, "fp8": 448.0}
CODE_BYTES = {"int4": 32, "fp4": 32, "int8": 64, "fp8": 64, "bf16": 128, "f32": 256}
FP4_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MAX_ROWS = 64 * 12 * 8192            # cached positions times heads of the largest attention call


def _attn(name, kv, B, NH, maxT, lens, fresh, page_rows):
    return {"name": name, "kind": "attn", "kv": kv, "B": B, "NH": NH, "maxT": maxT, "lens": lens, "fresh": fresh,
            "page_rows": page_rows}


def _verify(name, B, drafts, V, row, dtype, sure=False):
    return {"name": name, "kind": "verify", "B": B, "drafts": drafts, "V": V, "row": row, "dtype": dtype, "sure": sure}


def listed():
    """lens: > 0 the positions of every sequence, 0 per sequence ~ U[fresh, maxT].  fresh: new tokens
    a sequence, 1, or up to that many (0 among them).  page_rows 0: a contiguous cache."""
    return [
        # One user's token 1024, one layer: the smallest call, bound by latency.
        _attn("attn_fp4_T1024", "fp4", 1, 12, 1024, 1024, 1, 0),
        # 64 sequences of any length up to 8192: the largest call, bound by memory.
        _attn("attn_int4_ragged_8192", "int4", 64, 12, 8192, 0, 1, 256),
        # A serving batch with up to 7 drafts behind each last token.
        _attn("attn_fp4_drafts_b24", "fp4", 24, 12, 4096, 0, 8, 64),
        # Few sequences of a wide model with drafts, lengths that end inside a tile.
        _attn("attn_int4_drafts_b3", "int4", 3, 25, 1024, 999, 5, 64),
        # A batch of one length over a contiguous cache.
        _attn("attn_fp4_b16_T4096", "fp4", 16, 12, 4096, 4096, 1, 0),
        # The bookkeeping of a small decode step and of a step of many requests with prefill chunks
        # (some keep less than they held: refused drafts; some end).
        {"name": "tables_b24", "kind": "tables", "B": 24, "fresh": 8, "maxT": 4096, "page_rows": 64, "tight": False},
        {"name": "tables_b1000_prefill", "kind": "tables", "B": 1000, "fresh": 512, "maxT": 8192, "page_rows": 64,
         "tight": True},
        # K and V of a decode step with drafts, and of a prefill chunk.
        {"name": "rows_int4_t160", "kind": "rows", "kv": "int4", "tokens": 160, "NH": 12, "page_rows": 64},
        {"name": "rows_fp4_t8192", "kind": "rows", "kv": "fp4", "tokens": 8192, "NH": 12, "page_rows": 128},
        # One user's four drafts; a serving batch; drafts that come without probabilities (copied
        # from the prompt, say) against bf16 probabilities.
        _verify("verify_b1_k4", 1, 4, VOCAB, VOCAB_ROW, "f32"),
        _verify("verify_b64_k7", 64, 7, VOCAB, VOCAB_ROW, "f32"),
        _verify("verify_bf16_sure_b96_k3", 96, 3, VOCAB, VOCAB_ROW, "bf16", sure=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("attn", "attn", "attn", "tables", "rows", "verify"))
    if kind == "attn":
        B, NH = _log_int(rng, 1, 64), rng.choice((12, 12, rng.randint(1, 25)))
        paged = rng.random() < 0.7
        page_rows = rng.choice((64, 64, 128, 192, 256)) if paged else 0
        top = _log_int(rng, 64, min(8192, MAX_ROWS // (B * NH)))
        maxT = max(1, top // page_rows) * page_rows if paged else top
        fresh = rng.choice((1, rng.randint(2, 12))) if paged else 1
        lens = 0 if rng.random() < 0.6 else max(fresh, maxT - rng.randrange(maxT // 4 + 1))
        return {"kind": kind, "kv": rng.choice(("int4", "fp4")), "B": B, "NH": NH, "maxT": maxT, "lens": lens,
                "fresh": fresh, "page_rows": page_rows}
    if kind == "tables":
        return {"kind": kind, "B": _log_int(rng, 1, 1000), "fresh": _log_int(rng, 1, 512),
                "maxT": 256 * _log_int(rng, 4, 32), "page_rows": rng.choice((64, 128, 256)), "tight": rng.random() < 0.5}
    if kind == "rows":
        return {"kind": kind, "kv": rng.choice(("int4", "fp4", "int4", "fp4", "int8", "fp8", "bf16", "f32")),
                "tokens": _log_int(rng, 1, 8192), "NH": rng.choice((12, rng.randint(1, 12))),
                "page_rows": rng.choice((64, 128, 256))}
    V = rng.choice((VOCAB, _log_int(rng, 2, VOCAB)))
    return {"kind": kind, "B": _log_int(rng, 1, 64), "drafts": rng.randint(0, 7), "V": V,
            "row": VOCAB_ROW if V == VOCAB else V + rng.randint(0, 7), "dtype": rng.choice(("f32", "f32", "bf16")),
            "sure": rng.random() < 0.3}


# ------------------------------------------------------------------------------------
# Cache rows.
# ------------------------------------------------------------------------------------
def _act(kv):
    return torch.float32 if kv == "f32" else torch.bfloat16


def _encode(x, kv):
    """Rows of x [..., 64] (float) as stored bytes or elements, and their scales (None: no scale)."""
    if kv in ("bf16", "f32"):
        return x.to(_act(kv)), None
    scale = x.abs().amax(dim=-1) / LIMIT[kv]
    y = torch.where(scale.unsqueeze(-1) > 0, x / scale.unsqueeze(-1), torch.zeros_like(x))
    if kv == "int8":
        return y.round().clamp(-127, 127).to(torch.int8).view(torch.uint8), scale
    if kv == "fp8":
        return y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), scale
    if kv == "int4":
        nib = (y.round().clamp(-7, 7) + 8).to(torch.uint8)                 # code + 8
    else:
        a = y.abs()                                                         # nearest, ties to the even code
        mag = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
        nib = mag.to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)
    return nib[..., 0::2] | (nib[..., 1::2] << 4), scale                    # channel 2i in the low half of byte i


def _decode(stored, scale, kv, dtype):
    """Stored rows as values of `dtype`."""
    if kv in ("bf16", "f32"):
        return stored.to(dtype)
    if kv == "int8":
        v = stored.view(torch.int8).to(dtype)
    elif kv == "fp8":
        v = stored.view(torch.float8_e4m3fn).to(dtype)
    else:
        nib = torch.stack((stored & 15, stored >> 4), dim=-1).flatten(-2)
        if kv == "int4":
            v = nib.to(dtype) - 8
        else:
            table = torch.tensor(FP4_VALUES + tuple(-t for t in FP4_VALUES), dtype=dtype, device=stored.device)
            v = table[nib.long()]
    return v * scale.to(dtype).unsqueeze(-1)


class _Source:
    """Values of one seed, drawn in a fixed order."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def randn(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda")

    def rand(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")

    def ints(self, lo, hi, *shape):
        """int32 of lo .. hi."""
        return torch.randint(lo, hi + 1, shape, generator=self.g, device="cuda", dtype=torch.int32)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _counts(src, lo, hi, n):
    """n counts spread evenly over lo .. hi in an order of the seed's: their sum is the case's."""
    c = lo + torch.arange(n, device="cuda") * (hi - lo + 1) // n
    c[n - 1] = hi
    return c[src.perm(n)].to(torch.int32)


def _starts(fresh):
    start = torch.zeros(fresh.numel() + 1, dtype=torch.int32, device="cuda")
    start[1:] = torch.cumsum(fresh, 0)
    return start


# ------------------------------------------------------------------------------------
# Attention over a 4-bit cache.
# ------------------------------------------------------------------------------------
def _attn_inputs(case, seed):
    src, B, NH, maxT, kv = _Source(seed), case["B"], case["NH"], case["maxT"], case["kv"]
    fresh = _counts(src, 0 if case["fresh"] > 1 else 1, case["fresh"], B)
    lens = torch.full((B,), case["lens"], dtype=torch.int32, device="cuda")
    if not case["lens"]:
        lens = src.ints(min(case["fresh"], maxT), maxT, B)
    R = case["page_rows"] or maxT
    n = maxT // R
    pages = torch.empty((B * n, 2, NH, R, HD // 2), dtype=torch.uint8, device="cuda")
    scales = torch.empty((B * n, 2, NH, R), device="cuda")
    table = src.perm(B * n).to(torch.int32) if case["page_rows"] else torch.arange(B, dtype=torch.int32, device="cuda")
    step = max(1, (1 << 25) // (2 * NH * R * HD))
    for p0 in range(0, B * n, step):
        c, s = _encode(src.randn(min(step, B * n - p0), 2, NH, R, HD), kv)
        pages[p0:p0 + step], scales[p0:p0 + step] = c, s
    start = _starts(fresh)
    N = int(start[-1])
    # Heads of different sharpness.
    q = src.randn(N, 3, NH, HD) * (0.5 + 2 * src.rand(NH)).view(1, 1, NH, 1)
    return {"qkv": q.to(torch.bfloat16), "pages": pages, "scales": scales, "table": table.view(B, n), "start": start,
            "lens": lens, "starts": start.tolist(), "totals": lens.tolist()}


def _attn_prepare(case, seed):
    s = _attn_inputs(case, seed)
    B, NH, maxT = case["B"], case["NH"], case["maxT"]
    N = s["qkv"].shape[0]
    s["out"] = torch.zeros((N, NH, HD), dtype=torch.bfloat16, device="cuda")
    if own:
        from cuda_gpt2_inference_amd import kvattn
        s["ws"] = kvattn.Workspace(max(N, 1), NH, maxT)
        s["cur"] = s["lens"] - 1
        if case["page_rows"]:
            s["cache"] = kvattn.PagedCache(s["pages"], s["table"], s["table"].shape[1], case["page_rows"],
                                           s["pages"].shape[0], s["scales"])
        else:
            # [2][B][NH][maxT] rows: a contiguous cache keeps K of every sequence before V.
            s["kv"] = s["pages"].transpose(0, 1).contiguous()
            s["kvs"] = s["scales"].transpose(0, 1).contiguous()
    return s


def _attn_own(case, s):
    from cuda_gpt2_inference_amd import kvattn
    B, NH, maxT, kv = case["B"], case["NH"], case["maxT"], case["kv"]
    N = s["qkv"].shape[0]
    if N == 0:
        return s["out"]
    if not case["page_rows"]:
        kvattn.decode(s["out"], s["qkv"], s["kv"], B, NH, HD, maxT, kv_dtype=kv, kv_scale=s["kvs"], cur_len=s["cur"],
                      lens_per_seq=True, **s["ws"].kwargs())
    elif case["fresh"] == 1:
        kvattn.paged_decode(s["out"], s["qkv"], s["cache"], B, NH, HD, kv_dtype=kv, cur_len=s["cur"],
                            lens_per_seq=True, **s["ws"].kwargs())
    else:
        kvattn.paged_decode_tokens(s["out"], s["qkv"], s["cache"], s["start"], s["lens"], B, N, NH, HD, kv_dtype=kv,
                                   max_new=case["fresh"], **s["ws"].kwargs())
    return s["out"]


def _attn_plain(case, s):
    kv, starts = case["kv"], s["starts"]
    for b, T in enumerate(s["totals"]):
        t0, t1 = starts[b], starts[b + 1]
        if t1 == t0:
            continue
        R = s["pages"].shape[3]
        used = s["table"][b, :(T + R - 1) // R].long()
        # [pages, 2, NH, R, ...] -> [2, NH, T, ...]
        codes = s["pages"][used].permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :T]
        scale = s["scales"][used].permute(1, 2, 0, 3).flatten(2, 3)[:, :, :T]
        k, v = _decode(codes, scale, kv, torch.float32)
        q = s["qkv"][t0:t1, 0].float().transpose(0, 1).contiguous()         # [NH, n, HD]
        score = torch.matmul(q, k.transpose(1, 2).contiguous()) / 8.0
        n = t1 - t0
        seen = torch.arange(T, device="cuda").view(1, T) <= torch.arange(T - n, T, device="cuda").view(n, 1)
        score = score.masked_fill(~seen, float("-inf"))
        p = torch.exp(score - score.amax(dim=-1, keepdim=True))
        o = torch.matmul(p, v) / p.sum(dim=-1, keepdim=True)
        s["out"][t0:t1] = o.transpose(0, 1).to(torch.bfloat16)
    return s["out"]


def _attn_exact(case, seed):
    d = _attn_inputs(case, seed)
    R, kv = d["pages"].shape[3], case["kv"]
    out = torch.zeros((d["qkv"].shape[0], case["NH"], HD), dtype=torch.float64, device="cuda")
    for b, T in enumerate(d["totals"]):
        if d["starts"][b] == d["starts"][b + 1]:
            continue
        pos = torch.arange(T, device="cuda")
        at = (d["table"][b].long()[pos // R], pos % R)
        k, v = (_decode(d["pages"][at[0], part, :, at[1]], d["scales"][at[0], part, :, at[1]], kv, torch.float64)
                for part in (0, 1))                                          # [T, NH, HD]
        for t in range(d["starts"][b], d["starts"][b + 1]):
            seen = T - (d["starts"][b + 1] - t) + 1                         # positions up to this token's own
            w = torch.softmax((k[:seen] * d["qkv"][t, 0].double()).sum(-1) / math.sqrt(HD), dim=0)
            out[t] = (w.unsqueeze(-1) * v[:seen]).sum(0)
    return out


# ------------------------------------------------------------------------------------
# Block tables, token offsets and slot map.
# ------------------------------------------------------------------------------------
def _tables_prepare(case, seed):
    src, B, R, maxT = _Source(seed), case["B"], case["page_rows"], case["maxT"]
    n = maxT // R
    kept = src.ints(0, maxT - case["fresh"], B)
    fresh = src.ints(1, case["fresh"], B)
    kind = src.rand(B)
    held = kept.clone()
    held = torch.where(kind < 0.3, torch.clamp(kept + src.ints(0, 2 * R, B), max=maxT), held)   # refused drafts
    ended = kind > 0.95
    kept, fresh = (torch.where(ended, torch.zeros_like(kept), t) for t in (kept, fresh))
    new = kind.clone().gt(0.85) & ~ended                                    # requests that begin
    kept, held = (torch.where(new, torch.zeros_like(kept), t) for t in (kept, held))
    have, want = (held + R - 1) // R, (kept + fresh + R - 1) // R
    takes = int((want - have).clamp(min=0).sum())
    used, P = int(have.sum()), B * n
    free = takes // 2 if case["tight"] else min(takes + 7, P - used)
    ids = src.perm(P).to(torch.int32)
    table = torch.full((B, n), -1, dtype=torch.int32, device="cuda")
    first = torch.cumsum(have, 0) - have
    col = torch.arange(n, device="cuda", dtype=torch.int32)
    mine = col.view(1, n) < have.view(B, 1)
    table[mine] = ids[(first.view(B, 1) + col.view(1, n))[mine].long()]
    head = int(src.ints(0, P - 1, 1))
    pool = torch.full((4 + P,), -1, dtype=torch.int32, device="cuda")
    pool[:4] = torch.tensor([head, free, 0, 0], dtype=torch.int32)
    pool[4 + (head + torch.arange(free, device="cuda")) % P] = ids[used:used + free]
    N, room = int(fresh.sum()), B * case["fresh"]
    z = lambda k, t=torch.int32: torch.full((k,), -1, dtype=t, device="cuda")  # noqa: E731
    s = {"held": held, "kept": kept, "fresh": fresh, "table": table, "pool": pool, "P": P, "N": N, "room": room, "R": R,
         "held_out": z(B), "lens": z(B), "start": z(B + 1), "slots": z(room, torch.int64), "positions": z(room),
         "next": z(2)}
    if own:
        from cuda_gpt2_inference_amd import kvattn
        s["cache"] = kvattn.PagedCache(None, table, n, R, P)
    return s


def _tables_own(case, s):
    from cuda_gpt2_inference_amd import kvattn
    kvattn.paged_reserve(s["cache"], s["pool"], s["held"], s["kept"], s["fresh"], case["B"], held_out=s["held_out"],
                         lens=s["lens"], token_start=s["start"], slot_map=s["slots"], positions=s["positions"],
                         max_tokens=s["room"], pool_next=s["next"])
    return _tables_out(s)


def _tables_plain(case, s):
    R, P, N, n = s["R"], s["P"], s["N"], s["table"].shape[1]
    held, kept, fresh = s["held"].long(), s["kept"].long(), s["fresh"].long()
    head, count = s["pool"][0].long(), s["pool"][1].long()
    ring = s["pool"][4:]
    valid = (kept >= 0) & (kept <= held) & (held <= n * R) & (fresh >= 0) & (kept + fresh <= n * R)
    fresh = torch.where(valid, fresh, torch.zeros_like(fresh))
    have, want = (held + R - 1) // R, (kept + fresh + R - 1) // R
    takes = torch.where(valid, (want - have).clamp(min=0), torch.zeros_like(have))
    upto_takes, upto_tokens = torch.cumsum(takes, 0), torch.cumsum(fresh, 0)
    ok = valid & ((takes == 0) | (upto_takes <= count)) & ((fresh == 0) | (upto_tokens <= s["room"]))
    gives = torch.where(ok, (have - want).clamp(min=0), torch.zeros_like(have))
    took = torch.where(ok & (takes > 0), upto_takes, torch.zeros_like(takes)).amax()
    first = upto_takes - takes
    # Pages that go back to the ring, in request order.
    col = torch.arange(n, device="cuda").view(1, n)
    back = ok.view(-1, 1) & (col >= want.view(-1, 1)) & (col < have.view(-1, 1))
    freed = s["table"][back]
    ring[(head + count + torch.arange(freed.numel(), device="cuda")) % P] = freed
    # Pages that requests take.
    got = ok.view(-1, 1) & (col >= have.view(-1, 1)) & (col < want.view(-1, 1))
    at = (head + first.view(-1, 1) + col - have.view(-1, 1)) % P
    s["table"][got] = ring[at[got]]
    s["start"][0] = 0
    s["start"][1:] = upto_tokens
    s["held_out"].copy_(torch.where(ok, kept + fresh, held))
    s["lens"].copy_(torch.where(ok, kept + fresh, kept))
    s["next"][0] = (head + took) % P
    s["next"][1] = count - took + gives.sum()
    # Tokens.
    t = torch.arange(N, device="cuda")
    b = torch.searchsorted(upto_tokens, t, right=True)
    pos = kept[b] + t - (upto_tokens - fresh)[b]
    page = s["table"][b, pos // R].long()
    slot = torch.where(ok[b] & (page >= 0) & (page < P), page * R + pos % R, torch.full_like(pos, -1))
    s["slots"][:N] = slot
    s["positions"][:N] = pos
    return _tables_out(s)


def _tables_out(s):
    return {k: s[k] for k in ("table", "pool", "next", "held_out", "lens", "start", "slots", "positions")}


# ------------------------------------------------------------------------------------
# Rows by slot map.
# ------------------------------------------------------------------------------------
def _rows_inputs(case, seed):
    src, N, NH, R = _Source(seed), case["tokens"], case["NH"], case["page_rows"]
    P = N // R + 2
    qkv = (src.randn(N, 3, NH, HD) * torch.exp(src.randn(N, 3, NH, 1))).to(_act(case["kv"]))
    # Runs of neighbouring positions, as requests have them, over shuffled pages; every 50th or so
    # token is padding.
    pages = src.perm(P)
    pos = torch.arange(N, device="cuda") + int(src.ints(0, R, 1))
    slots = pages[(pos // R) % P] * R + pos % R
    slots[src.rand(N) < 0.02] = -1
    return {"qkv": qkv, "slots": slots, "P": P}


def _rows_prepare(case, seed):
    s = _rows_inputs(case, seed)
    N, NH, R, kv, P = case["tokens"], case["NH"], case["page_rows"], case["kv"], s["P"]
    store = _act(kv) if kv in ("bf16", "f32") else torch.uint8
    width = HD // 2 if kv in ("int4", "fp4") else HD
    s["pages"] = torch.zeros((P, 2, NH, R, width), dtype=store, device="cuda")
    s["scales"] = torch.zeros((P, 2, NH, R), device="cuda") if kv in LIMIT else None
    s["back"] = torch.zeros((N, 2, NH, HD), dtype=_act(kv), device="cuda")
    if own:
        from cuda_gpt2_inference_amd import kvattn
        s["cache"] = kvattn.PagedCache(s["pages"], None, 1, R, P, s["scales"])
    return s


def _rows_own(case, s):
    from cuda_gpt2_inference_amd import kvattn
    N, NH, kv = case["tokens"], case["NH"], case["kv"]
    kvattn.paged_store(s["cache"], s["qkv"], s["slots"], N, NH, HD, kv_dtype=kv)
    kvattn.paged_load(s["back"], s["cache"], s["slots"], N, NH, HD, kv_dtype=kv)
    return s["back"]


def _rows_plain(case, s):
    R, kv = case["page_rows"], case["kv"]
    there = (s["slots"] >= 0).nonzero().view(-1)
    page, row = s["slots"][there] // R, s["slots"][there] % R
    codes, scale = _encode(s["qkv"][there, 1:].float(), kv)
    s["pages"][page, :, :, row] = codes
    if scale is not None:
        s["scales"][page, :, :, row] = scale
        scale = s["scales"][page, :, :, row]
    s["back"][there] = _decode(s["pages"][page, :, :, row], scale, kv, torch.float32).to(_act(kv))
    return s["back"]


def _rows_exact(case, seed):
    d, kv = _rows_inputs(case, seed), case["kv"]
    x = d["qkv"][:, 1:]
    if kv in LIMIT:
        # The scale and the codes are what the type defines, a float and integers; their product in 64 bits.
        scale = (x.float().abs().amax(dim=-1, keepdim=True) / LIMIT[kv])
        y = torch.where(scale > 0, x.float() / scale, torch.zeros_like(scale))
        if kv == "fp4":
            grid = torch.tensor(FP4_VALUES, dtype=torch.float64, device="cuda")
            mids = ((grid[1:] + grid[:-1]) / 2).float()
            up = torch.bucketize(y.abs(), mids)                 # y on a middle: the lower value
            tie = (y.abs().unsqueeze(-1) == mids).any(-1) & (up % 2 == 1)
            code = grid[up + tie] * torch.sign(y).double()
        elif kv == "fp8":
            code = y.clamp(-448, 448).to(torch.float8_e4m3fn).double()
        else:
            code = y.double().round().clamp(-LIMIT[kv], LIMIT[kv])
        x = code * scale.double()
    return torch.where((d["slots"] >= 0).view(-1, 1, 1, 1), x.double(), torch.zeros((), dtype=torch.float64, device="cuda"))


# ------------------------------------------------------------------------------------
# Verification of drafted tokens.
# ------------------------------------------------------------------------------------
def _verify_prepare(case, seed):
    src, B, V, row = _Source(seed), case["B"], case["V"], case["row"]
    fresh = _counts(src, 1, case["drafts"] + 1, B)
    start = _starts(fresh)
    N = int(start[-1])
    dtype = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    p = torch.zeros((N, row), dtype=dtype, device="cuda")
    q = None if case["sure"] else torch.zeros((N, row), dtype=dtype, device="cuda")
    drafts = torch.empty(N, dtype=torch.int32, device="cuda")
    for t0 in range(0, N, 64):
        z = 2.5 * src.randn(min(64, N - t0), V)
        p[t0:t0 + 64, :V] = torch.softmax(z, dim=-1)
        zq = z + 0.7 * src.randn(*z.shape)
        if q is not None:
            q[t0:t0 + 64, :V] = torch.softmax(zq, dim=-1)
        # A draft is drawn from its own distribution; a sure one mostly is the likeliest token.
        noise = -torch.log(-torch.log(src.rand(*z.shape).clamp(1e-30, 1 - 1e-7)))
        drafts[t0:t0 + 64] = (zq + (0.1 if case["sure"] else 1.0) * noise).argmax(-1).to(torch.int32)
    s = {"p": p, "q": q, "drafts": drafts, "u": src.rand(N), "start": start, "N": N,
         "tokens": torch.full((N,), -1, dtype=torch.int32, device="cuda"),
         "count": torch.full((B,), -1, dtype=torch.int32, device="cuda")}
    if own:
        from cuda_gpt2_inference_amd import kvattn
        s["nbytes"] = kvattn.verify_workspace_bytes(B, V)
        s["ws"] = torch.empty(s["nbytes"], dtype=torch.uint8, device="cuda")
        kvattn.workspace_init(s["ws"], s["nbytes"])
    return s


def _verify_own(case, s):
    from cuda_gpt2_inference_amd import kvattn
    kvattn.verify_drafts(s["tokens"], s["count"], s["p"], s["drafts"], s["u"], s["start"], case["B"], s["N"], case["V"],
                         draft_probs=s["q"], row_stride=case["row"], dtype=case["dtype"], workspace=s["ws"],
                         workspace_nbytes=s["nbytes"])
    return {"tokens": s["tokens"], "count": s["count"]}


def _verify_plain(case, s):
    V, N, start = case["V"], s["N"], s["start"].long()
    first, last = start[:-1], start[1:] - 1
    t = torch.arange(N, device="cuda")
    x = s["drafts"].long()
    px = s["p"][t, x].double()
    qx = s["q"][t, x].double() if s["q"] is not None else torch.ones_like(px)
    accept = s["u"].double() * qx < px
    accept[last] = False                                            # a last row has no draft
    b = torch.searchsorted(start[1:], t, right=True)
    # The first row of every sequence that is not accepted: the row its next token is drawn from.
    row = torch.full((case["B"],), N, device="cuda").scatter_reduce(0, b, torch.where(accept, N, t), "amin")
    refused = row < last
    w = s["p"][row, :V].double()
    if s["q"] is not None:
        rest = w - torch.where(refused.view(-1, 1), s["q"][row, :V].double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    else:
        rest = w.clone()
        rest[refused, x[row][refused]] = 0.0
    rest = rest.clamp(min=0.0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, w)
    upto = torch.cumsum(rest, dim=-1)
    aim = s["u"].double()[last].view(-1, 1) * upto[:, -1:]          # a number that no draft was held against
    drawn = torch.searchsorted(upto, aim, right=True).view(-1)
    most = torch.where(rest > 0, torch.arange(V, device="cuda"), -1).amax(-1)
    drawn = torch.minimum(drawn, most)
    s["tokens"].copy_(torch.where(t < row[b], x, torch.where(t == row[b], drawn[b], -1)))
    s["count"].copy_(row - first + 1)
    return {"tokens": s["tokens"], "count": s["count"]}


# ------------------------------------------------------------------------------------
# The file's interface.
# ------------------------------------------------------------------------------------
def prepare(case, seed):
    make = {"attn": _attn_prepare, "tables": _tables_prepare, "rows": _rows_prepare, "verify": _verify_prepare}
    return {"case": case, **make[case["kind"]](case, seed)}


def run(state):
    case = state["case"]
    if own:
        call = {"attn": _attn_own, "tables": _tables_own, "rows": _rows_own, "verify": _verify_own}
    else:
        call = {"attn": _attn_plain, "tables": _tables_plain, "rows": _rows_plain, "verify": _verify_plain}
    return call[case["kind"]](case, state)


def exact(case, seed):
    """64-bit attention outputs and row values; tables and drawn tokens are whole numbers."""
    if case["kind"] == "rows":
        return _rows_exact(case, seed)
    return _attn_exact(case, seed) if case["kind"] == "attn" else None


def work(case):
    kind, B = case["kind"], case.get("B")
    if kind == "attn":
        T = case["lens"] or (case["maxT"] + 1) // 2                         # ragged: the mean
        n = 1 if case["fresh"] == 1 else case["fresh"] / 2
        return {"bytes": int(B * case["NH"] * (72 * T + n * 2 * 2 * HD)), "flops": int(B * case["NH"] * n * T * 4 * HD)}
    if kind == "tables":
        N = B * case["fresh"] // 2
        pages = B * case["fresh"] // (2 * case["page_rows"])
        return {"bytes": 24 * B + 12 * N + 8 * pages + 8, "flops": 0}
    if kind == "rows":
        act = 4 if case["kv"] == "f32" else 2
        row = CODE_BYTES[case["kv"]] + (4 if case["kv"] in LIMIT else 0)
        return {"bytes": case["tokens"] * (8 + 2 * case["NH"] * 2 * (HD * act + row)), "flops": 0}
    width = 4 if case["dtype"] == "f32" else 2
    rows = 1 if case["sure"] else 2
    return {"bytes": B * (case["V"] * width * rows + 16 * (case["drafts"] + 1)), "flops": 2 * B * case["V"]}
