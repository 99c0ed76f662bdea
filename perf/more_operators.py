"""The operators of a serving step that verifies a tree of drafted tokens, as timed cases.

Four kinds of case:

  tree    attention of a tree's tokens over a paged cache that holds their rows: every token sees the cached
          prefix, its ancestors and itself (``paged_decode_tree``), for every cache type
  walk    a step's tree: who sees whom and the tokens' positions from every token's parent (``tree_masks``), and
          the verification of the tree's tokens against the target's probabilities (``verify_tree``)
  logits  penalties for tokens that a sequence (and the row's branch of the tree) holds, biases and grammar masks,
          then logits or probabilities (``process_logits``)
  w4      a fully connected layer on 4-bit weights with a scale for every group of a row (``gemv_w4``)

With ``own`` the calls go to ``cuda_gpt2_inference_amd.kvattn``; without, they are computed with elementary torch
operations in 32 bits (sums of probabilities in 64).
"""
import math

import torch

own = False

HD = 64
VOCAB, VOCAB_ROW = 50257, 50304      # GPT-2's tokens, and the padded row of its logits
LIMIT = {"int4": 7.0, "fp4": 6.0, "int8": 127.0, "fp8": 448.0}
ROW_BYTES = {"int4": 36, "fp4": 36, "int8": 68, "fp8": 68, "bf16": 128, "f32": 256}     # of K or V, its scale with it
FP4_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MAX_ROWS = 16 * 12 * 8192            # cached positions times heads of the largest attention call
MAX_WEIGHTS = 50304 * 768            # weights of the largest layer


def _tree(name, kv, B, NH, maxT, lens, nodes, page_rows):
    return {"name": name, "kind": "tree", "kv": kv, "B": B, "NH": NH, "maxT": maxT, "lens": lens, "nodes": nodes,
            "page_rows": page_rows}


def _walk(name, B, nodes, V, row, dtype):
    return {"name": name, "kind": "walk", "B": B, "nodes": nodes, "V": V, "row": row, "dtype": dtype}


def _logits(name, B, nodes, V, row, dtype, out, probs, history, bias, grammar):
    return {"name": name, "kind": "logits", "B": B, "nodes": nodes, "V": V, "row": row, "dtype": dtype, "out": out,
            "probs": probs, "history": history, "bias": bias, "grammar": grammar}


def _w4(name, kind, B, M, K, group, out="bf16", gelu=False):
    return {"name": name, "kind": "w4", "codes": kind, "B": B, "M": M, "K": K, "group": group, "out": out, "gelu": gelu}


def listed():
    """lens: > 0 the positions of every sequence, 0 per sequence ~ U[nodes, maxT].  nodes: tokens of a sequence's tree,
    up to that many where there are several sequences (0 among them)."""
    return [
        # One user's tree of 26 drafts' tokens, one layer: the smallest call, bound by latency.
        _tree("tree_bf16_b1_n26", "bf16", 1, 12, 1024, 1000, 26, 64),
        # A serving batch over a 4-bit cache.
        _tree("tree_int4_b24_n32", "int4", 24, 12, 4096, 0, 32, 64),
        # Few sequences of a wide model, small trees, lengths that end inside a tile.
        _tree("tree_fp8_b3_n7", "fp8", 3, 25, 2048, 1999, 7, 128),
        # Long sequences with large trees over a cache of full width: the largest call.
        _tree("tree_bf16_b16_n64", "bf16", 16, 12, 8192, 0, 64, 256),
        # One user's tree; a serving batch, whose probabilities are kept in bf16.
        _walk("walk_b1_n26", 1, 26, VOCAB, VOCAB_ROW, "f32"),
        _walk("walk_bf16_b64_n16", 64, 16, VOCAB, VOCAB_ROW, "bf16"),
        # The rows of one user's tree with every rule; plain decoding of a batch; the logits alone, for a sampler
        # of the caller's.
        _logits("logits_b1_n26_probs", 1, 26, VOCAB, VOCAB_ROW, "f32", "f32", True, 900, 20, True),
        _logits("logits_b64_n1_probs", 64, 1, VOCAB, VOCAB_ROW, "f32", "f32", True, 2000, 0, True),
        _logits("logits_b32_n8", 32, 8, VOCAB, VOCAB_ROW, "bf16", "bf16", False, 4000, 50, False),
        # One token through the attention's output projection of GPT-2 medium; a tree's tokens through the up
        # projection of GPT-2 XL; a batch of trees through the vocabulary's table.
        _w4("w4_int4_1024x1024_b1", "int4", 1, 1024, 1024, 128),
        _w4("w4_fp4_6400x1600_b26", "fp4", 26, 6400, 1600, 32, gelu=True),
        _w4("w4_int4_vocabulary_b64", "int4", 64, 50304, 768, 64, out="f32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("tree", "tree", "walk", "logits", "logits", "w4", "w4"))
    if kind == "tree":
        B, NH = _log_int(rng, 1, 64), rng.choice((12, 12, rng.randint(1, 25)))
        page_rows = rng.choice((64, 64, 128, 192, 256))
        top = _log_int(rng, 128, min(8192, MAX_ROWS // (B * NH)))
        maxT = max(1, top // page_rows) * page_rows
        nodes = min(_log_int(rng, 1, 64), maxT)
        lens = 0 if rng.random() < 0.6 else max(nodes, maxT - rng.randrange(maxT // 4 + 1))
        kv = rng.choice(("int4", "fp4", "int8", "fp8", "bf16", "bf16", "f32"))
        if kv == "f32":
            B = max(1, min(B, MAX_ROWS // 2 // (NH * maxT)))
        return {"kind": kind, "kv": kv, "B": B, "NH": NH, "maxT": maxT, "lens": lens, "nodes": nodes,
                "page_rows": page_rows}
    if kind == "w4":
        B, group, K = _log_int(rng, 1, 64), rng.choice((32, 64, 128)), 64 * _log_int(rng, 2, 100)
        K = max(group, K // group * group)
        M = _log_int(rng, 16, min(50304, MAX_WEIGHTS // K))
        return {"kind": kind, "codes": rng.choice(("int4", "fp4")), "B": B, "M": M, "K": K, "group": group,
                "out": rng.choice(("bf16", "f32")), "gelu": rng.random() < 0.3}
    V = rng.choice((VOCAB, _log_int(rng, 2, VOCAB)))
    row = VOCAB_ROW if V == VOCAB else V + rng.randint(0, 7)
    B, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 32)
    nodes = max(1, min(nodes, 512 // B))
    if kind == "walk":
        return {"kind": kind, "B": B, "nodes": nodes, "V": V, "row": row, "dtype": rng.choice(("f32", "f32", "bf16"))}
    nodes = max(1, min(nodes, 128 // B))
    return {"kind": kind, "B": B, "nodes": nodes, "V": V, "row": row, "dtype": rng.choice(("f32", "bf16")),
            "out": rng.choice(("f32", "bf16")), "probs": rng.random() < 0.7, "history": _log_int(rng, 1, 8000),
            "bias": rng.choice((0, rng.randint(1, 300))), "grammar": rng.random() < 0.5}


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


def _dtype(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _sizes(src, n, most):
    """Tokens of each of n trees: `most` for one, else spread evenly over 0 .. most (1 where that is the most), in an
    order of the seed's."""
    if n == 1 or most == 1:
        return torch.full((n,), most, dtype=torch.int32, device="cuda")
    c = torch.arange(n, device="cuda") * (most + 1) // n
    c[n - 1] = most
    return c[src.perm(n)].to(torch.int32)


def _forest(src, sizes):
    """token_start, and every token's parent: the root first, then tokens behind one of the eight before."""
    start = torch.zeros(sizes.numel() + 1, dtype=torch.int32, device="cuda")
    start[1:] = torch.cumsum(sizes, 0)
    N = int(start[-1])
    t = torch.arange(N, device="cuda")
    owner = torch.searchsorted(start[1:].long(), t, right=True)
    at = t - start[owner].long()
    back = 1 + (src.rand(N) * torch.clamp(at, max=8)).long()
    parents = torch.where(at > 0, at - back.clamp(max=8), torch.full_like(at, -1))
    return start, owner, at, parents.clamp(min=-1).to(torch.int32)


def _sees(starts, parents, b):
    """[n, n] bool of tree b: row i sees token j (itself and its ancestors)."""
    t0, n = starts[b], starts[b + 1] - starts[b]
    p = parents[t0:t0 + n].long()
    sees = torch.eye(n, dtype=torch.bool, device="cuda")
    up = p.clone()
    rows = torch.arange(n, device="cuda")
    for _ in range(n):
        live = up >= 0
        sees[rows[live], up[live]] = True
        up = torch.where(live, p[up.clamp(min=0)], up)
    return sees


def _words(sees):
    """Bits of a bool matrix of up to 64 columns as one 64-bit word a row."""
    n = sees.shape[1]
    bit = torch.ones(n, dtype=torch.int64, device="cuda") << torch.arange(n, device="cuda")
    return (sees.to(torch.int64) * bit).sum(-1)


# ------------------------------------------------------------------------------------
# Attention of a tree's tokens.
# ------------------------------------------------------------------------------------
def _encode(x, kv):
    """Rows of x [..., 64] (float) as stored bytes or elements, and their scales (None: no scale)."""
    if kv in ("bf16", "f32"):
        return x.to(_dtype(kv)), None
    scale = x.abs().amax(dim=-1) / LIMIT[kv]
    y = torch.where(scale.unsqueeze(-1) > 0, x / scale.unsqueeze(-1), torch.zeros_like(x))
    if kv == "int8":
        return y.round().clamp(-127, 127).to(torch.int8).view(torch.uint8), scale
    if kv == "fp8":
        return y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), scale
    nib = _nibbles(y, kv)
    return nib[..., 0::2] | (nib[..., 1::2] << 4), scale                    # channel 2i in the low half of byte i


def _nibbles(y, kind):
    """4-bit codes of y, already divided by its scale."""
    if kind == "int4":
        return (y.round().clamp(-7, 7) + 8).to(torch.uint8)
    a = y.abs()                                                             # nearest, ties to the even code
    mag = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    return mag.to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)


def _codes(packed, kind, dtype):
    """The numbers that packed 4-bit codes stand for, without their scales."""
    nib = torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2)
    if kind == "int4":
        return nib.to(dtype) - 8
    return torch.tensor(FP4_VALUES + tuple(-t for t in FP4_VALUES), dtype=dtype, device=packed.device)[nib.long()]


def _decode(stored, scale, kv, dtype):
    """Stored rows as values of `dtype`."""
    if kv in ("bf16", "f32"):
        return stored.to(dtype)
    if kv == "int8":
        v = stored.view(torch.int8).to(dtype)
    elif kv == "fp8":
        v = stored.view(torch.float8_e4m3fn).to(dtype)
    else:
        v = _codes(stored, kv, dtype)
    return v * scale.to(dtype).unsqueeze(-1)


def _tree_inputs(case, seed):
    src, B, NH, maxT, kv = _Source(seed), case["B"], case["NH"], case["maxT"], case["kv"]
    start, owner, at, parents = _forest(src, _sizes(src, B, case["nodes"]))
    lens = torch.full((B,), case["lens"], dtype=torch.int32, device="cuda")
    if not case["lens"]:
        lens = src.ints(min(case["nodes"], maxT), maxT, B)
    R = case["page_rows"]
    n = maxT // R
    width = HD // 2 if kv in ("int4", "fp4") else HD
    store = _dtype(kv) if kv in ("bf16", "f32") else torch.uint8
    pages = torch.empty((B * n, 2, NH, R, width), dtype=store, device="cuda")
    scales = torch.empty((B * n, 2, NH, R), device="cuda") if kv in LIMIT else None
    step = max(1, (1 << 25) // (2 * NH * R * HD))
    for p0 in range(0, B * n, step):
        c, s = _encode(src.randn(min(step, B * n - p0), 2, NH, R, HD), kv)
        pages[p0:p0 + step] = c
        if scales is not None:
            scales[p0:p0 + step] = s
    starts = start.tolist()
    # Heads of different sharpness.
    q = src.randn(starts[-1], 3, NH, HD) * (0.5 + 2 * src.rand(NH)).view(1, 1, NH, 1)
    return {"qkv": q.to(_dtype("f32" if kv == "f32" else "bf16")), "pages": pages, "scales": scales,
            "table": src.perm(B * n).to(torch.int32).view(B, n), "start": start, "parents": parents, "lens": lens,
            "starts": starts, "totals": lens.tolist()}


def _tree_prepare(case, seed):
    s = _tree_inputs(case, seed)
    NH, maxT = case["NH"], case["maxT"]
    N = s["starts"][-1]
    s["out"] = torch.zeros((N, NH, HD), dtype=s["qkv"].dtype, device="cuda")
    # Who sees whom: made once a step, read by every layer.
    sees = [_sees(s["starts"], s["parents"], b) for b in range(case["B"])]
    s["sees"] = sees
    s["masks"] = torch.cat([_words(x) for x in sees]).view(N, 1)
    if own:
        from cuda_gpt2_inference_amd import kvattn
        s["ws"] = kvattn.Workspace(max(N, 1), NH, maxT)
        s["cache"] = kvattn.PagedCache(s["pages"], s["table"], s["table"].shape[1], case["page_rows"],
                                       s["pages"].shape[0], s["scales"])
    return s


def _tree_own(case, s):
    from cuda_gpt2_inference_amd import kvattn
    N = s["starts"][-1]
    if N:
        kvattn.paged_decode_tree(s["out"], s["qkv"], s["cache"], s["start"], s["lens"], s["masks"], case["B"], N,
                                 case["NH"], HD, kv_dtype=case["kv"], max_new=case["nodes"], **s["ws"].kwargs())
    return s["out"]


def _tree_plain(case, s):
    kv, starts = case["kv"], s["starts"]
    for b, T in enumerate(s["totals"]):
        t0, t1 = starts[b], starts[b + 1]
        n = t1 - t0
        if n == 0:
            continue
        R = s["pages"].shape[3]
        used = s["table"][b, :(T + R - 1) // R].long()
        # [pages, 2, NH, R, ...] -> [2, NH, T, ...]
        codes = s["pages"][used].permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :T]
        scale = s["scales"][used].permute(1, 2, 0, 3).flatten(2, 3)[:, :, :T] if s["scales"] is not None else None
        k, v = _decode(codes, scale, kv, torch.float32)
        q = s["qkv"][t0:t1, 0].float().transpose(0, 1).contiguous()         # [NH, n, HD]
        score = torch.matmul(q, k.transpose(1, 2).contiguous()) / 8.0
        seen = torch.ones((n, T), dtype=torch.bool, device="cuda")
        seen[:, T - n:] = s["sees"][b]
        score = score.masked_fill(~seen, float("-inf"))
        p = torch.exp(score - score.amax(dim=-1, keepdim=True))
        o = torch.matmul(p, v.contiguous()) / p.sum(dim=-1, keepdim=True)
        s["out"][t0:t1] = o.transpose(0, 1).to(s["out"].dtype)
    return s["out"]


def _tree_exact(case, seed):
    d = _tree_inputs(case, seed)
    R, kv = d["pages"].shape[3], case["kv"]
    out = torch.zeros((d["starts"][-1], case["NH"], HD), dtype=torch.float64, device="cuda")
    parents = d["parents"].tolist()
    for b, T in enumerate(d["totals"]):
        t0, t1 = d["starts"][b], d["starts"][b + 1]
        if t0 == t1:
            continue
        pos = torch.arange(T, device="cuda")
        page, row = d["table"][b].long()[pos // R], pos % R
        k, v = (_decode(d["pages"][page, part, :, row], None if d["scales"] is None else d["scales"][page, part, :, row],
                        kv, torch.float64).transpose(0, 1).contiguous() for part in (0, 1))     # [NH, T, HD]
        for t in range(t0, t1):
            mine = list(range(T - (t1 - t0)))                               # the prefix, then the token's branch
            i = t - t0
            while i >= 0:
                mine.append(T - (t1 - t0) + i)
                i = parents[t0 + i]
            mine = torch.tensor(mine, device="cuda")
            kk, vv = k[:, mine], v[:, mine]
            w = torch.softmax((kk * d["qkv"][t, 0].double().unsqueeze(1)).sum(-1) / math.sqrt(HD), dim=-1)
            out[t] = (w.unsqueeze(-1) * vv).sum(1)
    return out


# ------------------------------------------------------------------------------------
# A step's tree and its verification.
# ------------------------------------------------------------------------------------
def _walk_prepare(case, seed):
    src, B, V, row = _Source(seed), case["B"], case["V"], case["row"]
    start, owner, at, parents = _forest(src, _sizes(src, B, case["nodes"]))
    N = int(start[-1])
    p = torch.zeros((N, row), dtype=_dtype(case["dtype"]), device="cuda")
    for t0 in range(0, N, 64):
        p[t0:t0 + 64, :V] = torch.softmax(2.5 * src.randn(min(64, N - t0), V), dim=-1)
    # A token is one of the likelier behind its parent.
    tokens = src.ints(0, V - 1, N)
    from_row = (start[owner] + parents.clamp(min=0)).long()
    for t0 in range(0, N, 64):
        z = torch.log(p[from_row[t0:t0 + 64], :V].float().clamp(min=1e-30))
        noise = -torch.log(-torch.log(src.rand(*z.shape).clamp(1e-30, 1 - 1e-7)))
        tokens[t0:t0 + 64] = (2.0 * z + noise).argmax(-1).to(torch.int32)
    i32 = lambda *s: torch.full(s, -1, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"p": p, "tree": tokens, "parents": parents, "start": start, "owner": owner, "at": at, "from_row": from_row,
         "u": src.rand(N), "draw": src.rand(B), "lens": src.ints(case["nodes"], 8000, B), "N": N,
         "masks": torch.zeros((N, 1), dtype=torch.int64, device="cuda"), "positions": i32(N), "tokens": i32(N),
         "path": i32(N), "counts": i32(B), "kept": i32(B)}
    if own:
        from cuda_gpt2_inference_amd import kvattn
        s["nbytes"] = kvattn.verify_workspace_bytes(B, V)
        s["ws"] = torch.empty(s["nbytes"], dtype=torch.uint8, device="cuda")
        kvattn.workspace_init(s["ws"], s["nbytes"])
    return s


def _walk_out(s):
    return {k: s[k] for k in ("masks", "positions", "tokens", "path", "counts", "kept")}


def _walk_own(case, s):
    from cuda_gpt2_inference_amd import kvattn
    B, N = case["B"], s["N"]
    kvattn.tree_masks(s["masks"], s["parents"], s["start"], B, N, positions=s["positions"], lens=s["lens"])
    kvattn.verify_tree(s["tokens"], s["path"], s["counts"], s["p"], s["tree"], s["parents"], s["u"], s["draw"], s["start"], B,
                       N, case["V"], lens=s["lens"], kept=s["kept"], row_stride=case["row"], dtype=case["dtype"],
                       workspace=s["ws"], workspace_nbytes=s["nbytes"])
    return _walk_out(s)


def _walk_plain(case, s):
    B, N, V, n = case["B"], s["N"], case["V"], case["nodes"]
    owner, at, start = s["owner"], s["at"], s["start"].long()
    sizes = start[1:] - start[:-1]
    col = torch.arange(n, device="cuda")
    # Token rows as [B, n], the places past a tree's end marked.
    real = col.view(1, n) < sizes.view(B, 1)
    row = torch.where(real, start[:-1].view(B, 1) + col.view(1, n), 0)
    par = torch.where(real, s["parents"].long()[row], torch.full_like(row, -2))
    # Masks and positions: one generation after another.
    sees = torch.eye(n, dtype=torch.bool, device="cuda").repeat(B, 1, 1)
    up = par.clone()
    depth = torch.zeros_like(par)
    for _ in range(n):
        live = up >= 0
        sees |= live.unsqueeze(-1) & (up.unsqueeze(-1) == col.view(1, 1, n))
        depth += live
        up = torch.where(live, torch.gather(par, 1, up.clamp(min=0)), up)
    bit = torch.ones(n, dtype=torch.int64, device="cuda") << col
    s["masks"][:, 0] = (sees.to(torch.int64) * bit.view(1, 1, n)).sum(-1)[owner, at]
    s["positions"].copy_(((s["lens"].long() - sizes).view(B, 1) + depth).clamp(min=0)[owner, at])
    # Mass of every token behind its parent; a token that an earlier child of the parent is has none left.
    x = s["tree"].long()
    mass = torch.where((s["parents"] >= 0), s["p"][s["from_row"], x].double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    mass = torch.where(real, mass[row], torch.zeros((), dtype=torch.float64, device="cuda"))
    tok = x[row]
    before = (par.unsqueeze(2) == par.unsqueeze(1)) & (col.view(1, 1, n) < col.view(1, n, 1)) & real.unsqueeze(1)
    again = (before & (tok.unsqueeze(2) == tok.unsqueeze(1))).any(-1)
    mass = torch.where(again, torch.zeros_like(mass), mass)
    low = (before.double() * mass.unsqueeze(1)).sum(-1)
    u = s["u"].double()[s["from_row"]][row]
    chosen = real & (par >= 0) & (u >= low) & (u < low + mass)
    # The walk.
    on = torch.zeros((B, n), dtype=torch.bool, device="cuda")
    on[:, 0] = real[:, 0]
    for i in range(1, n):
        on[:, i] = chosen[:, i] & torch.gather(on, 1, par[:, i:i + 1].clamp(min=0)).view(B)
    some = sizes > 0
    last = torch.where(on, col.view(1, n), -1).amax(-1)
    steps = on.sum(-1)                                              # tokens on the path, the root among them
    # What is left of the last row is drawn from.
    w = s["p"][(start[:-1] + last.clamp(min=0)).clamp(max=N - 1), :V].double()
    left = w.clone()
    child = real & (par == last.view(B, 1))
    b = torch.arange(B, device="cuda").view(B, 1).expand(B, n)
    left[b[child], tok[child]] = 0.0
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, w)
    upto = torch.cumsum(left, dim=-1)
    drawn = torch.searchsorted(upto, s["draw"].double().view(B, 1) * upto[:, -1:], right=True).view(-1)
    drawn = torch.minimum(drawn, torch.where(left > 0, torch.arange(V, device="cuda"), -1).amax(-1))
    # Path first, -1 behind; the accepted tokens are the path's without its root, then the drawn one.
    order = torch.argsort(torch.where(on, col.view(1, n), n + col.view(1, n)), dim=-1)
    path = torch.where(col.view(1, n) < steps.view(B, 1), order, -1)
    out = torch.roll(torch.gather(tok, 1, order), -1, dims=1)
    out = torch.where(col.view(1, n) < steps.view(B, 1) - 1, out, -1)
    out = torch.where(col.view(1, n) == steps.view(B, 1) - 1, drawn.view(B, 1), out)
    s["path"].copy_(path[owner, at])
    s["tokens"].copy_(out[owner, at])
    s["counts"].copy_(torch.where(some, steps, 0))
    s["kept"].copy_(s["lens"].long() - sizes + steps)
    return _walk_out(s)


# ------------------------------------------------------------------------------------
# Penalties, biases and grammar masks on logits.
# ------------------------------------------------------------------------------------
def _logits_inputs(case, seed):
    src, B, V, row = _Source(seed), case["B"], case["V"], case["row"]
    start, owner, at, parents = _forest(src, _sizes(src, B, case["nodes"]))
    N = int(start[-1])
    x = torch.zeros((N, row), dtype=_dtype(case["dtype"]), device="cuda")
    x[:, :V] = 2.5 * src.randn(N, V)
    most = case["history"]
    d = {"x": x, "start": start, "owner": owner, "at": at, "parents": parents, "N": N,
         # Text repeats its common tokens.
         "history": (V * src.rand(B, most) ** 4).to(torch.int32).clamp(max=V - 1),
         "held": src.ints(most // 2, most, B), "tree": (V * src.rand(N) ** 4).to(torch.int32).clamp(max=V - 1),
         "repetition": 1.0 + 0.3 * src.rand(B), "frequency": 0.5 * src.rand(B), "presence": 0.5 * src.rand(B),
         # Every seventh sequence or so takes the likeliest token.
         "temperature": torch.where(src.rand(B) < 0.15, torch.zeros(B, device="cuda"), 0.6 + 0.8 * src.rand(B)),
         "starts": start.tolist()}
    d["prompt"] = (d["held"] * src.rand(B)).to(torch.int32)
    n = case["bias"]
    if n:
        count = src.ints(0, n, B)
        d["bias_start"] = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
        d["bias_start"][1:] = torch.cumsum(count, 0)
        m = int(d["bias_start"][-1])
        d["bias_ids"], d["bias"] = src.ints(0, V - 1, m), 3.0 * src.randn(m)
    if case["grammar"]:
        # A few grammars' states: some allow most of the tokens, some few; a fifth of the rows have none.
        states = 5
        d["allowed"] = torch.zeros((states, (V + 31) // 32), dtype=torch.int32, device="cuda")
        for i in range(states):
            ok = src.rand((V + 31) // 32, 32) < (0.95, 0.5, 0.1, 0.01, 0.9)[i]
            bit = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
            w = (ok.to(torch.int64) * bit).sum(-1)
            d["allowed"][i] = torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)
        d["allowed_of"] = src.ints(-1, states - 1, N)
    return d


def _logits_prepare(case, seed):
    s = _logits_inputs(case, seed)
    N = s["N"]
    s["out"] = torch.zeros((N, case["row"]), dtype=_dtype(case["out"]), device="cuda")
    s["sees"] = [_sees(s["starts"], s["parents"], b) for b in range(case["B"])]
    if own:
        from cuda_gpt2_inference_amd import kvattn
        s["masks"] = torch.cat([_words(x) for x in s["sees"]]).view(N, 1)
        rules = {"repetition": s["repetition"], "frequency": s["frequency"], "presence": s["presence"],
                 "history": s["history"], "history_len": s["held"], "prompt_len": s["prompt"],
                 "max_history": case["history"], "tokens": s["tree"], "masks": s["masks"], "mask_words": 1}
        if case["probs"]:
            rules["temperature"] = s["temperature"]
        if case["bias"]:
            rules.update(bias_start=s["bias_start"], bias_ids=s["bias_ids"], bias=s["bias"],
                         num_bias=s["bias_ids"].numel(), max_bias=case["bias"])
        if case["grammar"]:
            rules.update(allowed=s["allowed"], allowed_of=s["allowed_of"], num_allowed=s["allowed"].shape[0],
                         allowed_stride=s["allowed"].shape[1])
        s["rules"] = kvattn.LogitRules(**rules)
    return s


def _logits_own(case, s):
    from cuda_gpt2_inference_amd import kvattn
    kvattn.process_logits(s["out"], s["x"], s["rules"], s["start"], case["B"], s["N"], case["V"], row_stride=case["row"],
                          out_stride=case["row"], dtype=case["dtype"], out_dtype=case["out"], probs=case["probs"])
    return s["out"]


def _logits_plain(case, s):
    B, V, N = case["B"], case["V"], s["N"]
    owner = s["owner"]
    place = torch.arange(case["history"], device="cuda").view(1, -1)
    there = (place < s["held"].view(B, 1)).float()
    made = there * (place >= s["prompt"].view(B, 1))
    ids = s["history"].long()
    seen = torch.zeros((B, V), device="cuda").scatter_add_(1, ids, there)[owner]
    count = torch.zeros((B, V), device="cuda").scatter_add_(1, ids, made)[owner]
    for b in range(B):
        t0, t1 = s["starts"][b], s["starts"][b + 1]
        if t1 > t0:
            tok = s["tree"][t0:t1].long().view(1, -1).expand(t1 - t0, -1)
            branch = torch.zeros((t1 - t0, V), device="cuda").scatter_add_(1, tok, s["sees"][b].float())
            seen[t0:t1] += branch
            count[t0:t1] += branch
    x = s["x"][:, :V].float()
    r = s["repetition"][owner].view(N, 1)
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - (s["frequency"][owner].view(N, 1) * count + s["presence"][owner].view(N, 1) * (count > 0))
    if case["bias"]:
        # Of an id that is listed twice the last entry holds.
        m = s["bias_ids"].numel()
        of = torch.searchsorted(s["bias_start"][1:].long(), torch.arange(m, device="cuda"), right=True)
        entry = torch.full((B * V,), -1, dtype=torch.int64, device="cuda")
        entry.scatter_reduce_(0, of * V + s["bias_ids"].long(), torch.arange(m, device="cuda"), "amax")
        entry = entry.view(B, V)[owner]
        if m:
            x = torch.where(entry >= 0, x + s["bias"][entry.clamp(min=0)], x)
    if case["grammar"]:
        v = torch.arange(V, device="cuda")
        of = s["allowed_of"].long()
        ok = (s["allowed"][of.clamp(min=0)][:, v // 32] >> (v % 32).to(torch.int32)) & 1
        x = x.masked_fill((ok == 0) & (of >= 0).view(N, 1), float("-inf"))
    if case["probs"]:
        t = s["temperature"][owner].view(N, 1)
        top = x.amax(-1, keepdim=True)
        e = torch.exp((x - top) / torch.where(t > 0, t, torch.ones_like(t)))
        first = torch.where(x == top, torch.arange(V, device="cuda"), V).amin(-1, keepdim=True)
        one = (torch.arange(V, device="cuda") == first).float()
        x = torch.where(t > 0, e / e.sum(-1, keepdim=True), one)
        x = torch.where(top == float("-inf"), torch.zeros_like(x), x)
    s["out"][:, :V] = x.to(s["out"].dtype)
    return s["out"]


def _logits_exact(case, seed):
    d = _logits_inputs(case, seed)
    B, V, N = case["B"], case["V"], d["N"]
    out = torch.zeros((N, case["row"]), dtype=torch.float64, device="cuda")
    owner, parents, starts = d["owner"].tolist(), d["parents"].tolist(), d["starts"]
    held, prompt, states = d["held"].tolist(), d["prompt"].tolist(), d["allowed_of"].tolist() if case["grammar"] else None
    bias_start = d["bias_start"].tolist() if case["bias"] else None
    value = {k: d[k].double() for k in ("repetition", "frequency", "presence", "temperature")}
    for t in range(N):
        b = owner[t]
        branch, i = [], t - starts[b]
        while i >= 0:
            branch.append(starts[b] + i)
            i = parents[starts[b] + i]
        branch = d["tree"][torch.tensor(branch, device="cuda")].long()
        made = torch.cat((d["history"][b, prompt[b]:held[b]].long(), branch))
        count = torch.bincount(made, minlength=V).double()
        held_at_all = torch.bincount(torch.cat((d["history"][b, :held[b]].long(), branch)), minlength=V) > 0
        x = d["x"][t, :V].double()
        x = torch.where(held_at_all, torch.where(x > 0, x / value["repetition"][b], x * value["repetition"][b]), x)
        x = x - value["frequency"][b] * count - torch.where(count > 0, value["presence"][b], torch.zeros_like(x))
        if bias_start:
            lo, hi = bias_start[b], bias_start[b + 1]
            last = dict(zip(d["bias_ids"][lo:hi].tolist(), range(lo, hi)))
            if last:
                x[torch.tensor(list(last), device="cuda")] += d["bias"][torch.tensor(list(last.values()), device="cuda")].double()
        if states and states[t] >= 0:
            v = torch.arange(V, device="cuda")
            ok = (d["allowed"][states[t]].long()[v // 32] >> (v % 32)) % 2 != 0
            x[~ok] = float("-inf")
        if case["probs"]:
            top = x.max()
            if top == float("-inf"):
                x = torch.zeros_like(x)
            elif value["temperature"][b] > 0:
                x = torch.softmax(x / value["temperature"][b], dim=0)
            else:
                x = (torch.arange(V, device="cuda") == (x == top).nonzero()[0, 0]).double()
        out[t, :V] = x
    return out


# ------------------------------------------------------------------------------------
# Fully connected layers on 4-bit weights.
# ------------------------------------------------------------------------------------
def _w4_inputs(case, seed):
    src, B, M, K, G = _Source(seed), case["B"], case["M"], case["K"], case["group"]
    w = (src.randn(M, K // G, G) * (0.02 * torch.exp(0.3 * src.randn(M, K // G, 1))))
    scale = (w.abs().amax(-1) / LIMIT[case["codes"]]).to(torch.bfloat16)
    nib = _nibbles(w / scale.float().clamp(min=1e-30).unsqueeze(-1), case["codes"]).view(M, K)
    return {"codes": nib[:, 0::2] | (nib[:, 1::2] << 4), "scale": scale,        # column 2i in the low half of byte i
            "x": src.randn(B, K).to(torch.bfloat16), "bias": (0.1 * src.randn(M)).to(torch.bfloat16)}


def _w4_prepare(case, seed):
    s = _w4_inputs(case, seed)
    s["out"] = torch.zeros((case["B"], case["M"]), dtype=_dtype(case["out"]), device="cuda")
    if own:
        from cuda_gpt2_inference_amd import kvattn
        s["w4"] = kvattn.w4_pack(s["codes"], s["scale"], case["M"], case["K"], case["group"], w_dtype=case["codes"])
    return s


def _w4_own(case, s):
    from cuda_gpt2_inference_amd import kvattn
    kvattn.gemv_w4(s["out"], s["w4"], s["x"], case["B"], case["M"], case["K"], group=case["group"], w_dtype=case["codes"],
                   bias=s["bias"], out_dtype=case["out"], gelu=case["gelu"])
    return s["out"]


def _w4_plain(case, s):
    M, K, G = case["M"], case["K"], case["group"]
    w = (_codes(s["codes"], case["codes"], torch.float32).view(M, K // G, G) * s["scale"].float().unsqueeze(-1)).view(M, K)
    y = torch.matmul(s["x"].float(), w.t()) + s["bias"].float()
    if case["gelu"]:
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    s["out"].copy_(y.to(s["out"].dtype))
    return s["out"]


def _w4_exact(case, seed):
    d = _w4_inputs(case, seed)
    out = torch.empty((case["B"], case["M"]), dtype=torch.float64, device="cuda")
    x = d["x"].double()
    for m0 in range(0, case["M"], 4096):
        code = _codes(d["codes"][m0:m0 + 4096], case["codes"], torch.float64)
        w = code * d["scale"][m0:m0 + 4096].double().repeat_interleave(case["group"], dim=1)
        out[:, m0:m0 + 4096] = x @ w.t().contiguous() + d["bias"][m0:m0 + 4096].double()
    if case["gelu"]:
        out = 0.5 * out * (1 + torch.tanh(math.sqrt(2 / math.pi) * (out + 0.044715 * out ** 3)))
    return out


# ------------------------------------------------------------------------------------
# The file's interface.
# ------------------------------------------------------------------------------------
def prepare(case, seed):
    make = {"tree": _tree_prepare, "walk": _walk_prepare, "logits": _logits_prepare, "w4": _w4_prepare}
    return {"case": case, **make[case["kind"]](case, seed)}


def run(state):
    case = state["case"]
    if own:
        call = {"tree": _tree_own, "walk": _walk_own, "logits": _logits_own, "w4": _w4_own}
    else:
        call = {"tree": _tree_plain, "walk": _walk_plain, "logits": _logits_plain, "w4": _w4_plain}
    return call[case["kind"]](case, state)


def exact(case, seed):
    """In 64 bits; masks, paths and drawn tokens are whole numbers."""
    make = {"tree": _tree_exact, "logits": _logits_exact, "w4": _w4_exact}
    return make[case["kind"]](case, seed) if case["kind"] in make else None


def work(case):
    kind, B = case["kind"], case["B"]
    if kind == "w4":
        M, K = case["M"], case["K"]
        return {"bytes": M * K // 2 + 2 * M * K // case["group"] + 2 * (B * K + M) + B * M * (4 if case["out"] == "f32" else 2),
                "flops": 2 * B * M * K}
    n = case["nodes"] if B == 1 or case["nodes"] == 1 else case["nodes"] / 2
    if kind == "tree":
        T = case["lens"] or (case["nodes"] + case["maxT"]) // 2              # ragged: the mean
        act = 4 if case["kv"] == "f32" else 2
        return {"bytes": int(B * case["NH"] * (2 * ROW_BYTES[case["kv"]] * T + n * 2 * act * HD)),
                "flops": int(B * case["NH"] * n * T * 4 * HD)}
    width = {"f32": 4, "bf16": 2}
    if kind == "walk":
        return {"bytes": int(B * (case["V"] * width[case["dtype"]] + 40 * n)), "flops": 2 * B * case["V"]}
    rules = B * (case["history"] * 3 + case["bias"] * 4) + (5 * case["V"] // 8 if case["grammar"] else 0)
    return {"bytes": int(B * n * case["V"] * (width[case["dtype"]] + width[case["out"]]) + rules),
            "flops": int(8 * B * n * case["V"])}
