"""Plain restatements, in 64 bits, of what a step with trees of drafted tokens does, and the bounds that the tests
hold the kernels to."""
import math

import numpy as np

import kv4ref

HS = 64
LOG2E = 1.4426950408889634
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}


def bf16(x):
    """float32 array rounded to bf16, as float32."""
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16).float().numpy()


def forest(r, sizes, wild=False):
    """token_start and parents of trees of the given sizes; wild: some parents that count as none."""
    start = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    parents = np.full(start[-1], -1, dtype=np.int32)
    for t0, n in zip(start, sizes):
        for i in range(1, n):
            parents[t0 + i] = r.randint(max(0, i - 6), i)
            if wild and r.rand() < 0.1:
                parents[t0 + i] = r.choice([-7, i, i + 1, n, 1 << 30])
    return start, parents


def branch(parents, t0, i):
    """Indices of token i and its ancestors."""
    out = []
    while i >= 0:
        out.append(i)
        p = int(parents[t0 + i])
        i = p if 0 <= p < i else -1
    return out


def masks(start, parents, words):
    out = np.zeros((len(parents), words), dtype=np.uint64)
    depth = np.zeros(len(parents), dtype=np.int64)
    for t0, t1 in zip(start[:-1], start[1:]):
        for i in range(t1 - t0):
            if i < 64 * words:
                b = branch(parents, t0, i)
                depth[t0 + i] = len(b) - 1
                for j in b:
                    out[t0 + i, j >> 6] |= np.uint64(1 << (j & 63))
    return out, depth


# ------------------------------------------------------------------------------------
# Cache rows of every type.
# ------------------------------------------------------------------------------------
def encode(x, kv):
    """Rows x [..., 64] -> stored torch tensor, scales (None: none)."""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32))
    if kv == "f32":
        return t, None
    if kv == "bf16":
        return t.to(torch.bfloat16), None
    if kv in ("int4", "fp4"):
        codes, scale = kv4ref.encode(x, kv)
        return torch.from_numpy(codes), torch.from_numpy(scale)
    scale = t.abs().amax(-1) / (127.0 if kv == "int8" else 448.0)
    y = torch.where(scale.unsqueeze(-1) > 0, t / scale.unsqueeze(-1), torch.zeros_like(t))
    if kv == "int8":
        return y.round().clamp(-127, 127).to(torch.int8).view(torch.uint8), scale
    return y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), scale


def decode(stored, scale, kv):
    """-> values in 64 bits (numpy)."""
    import torch
    if kv in ("f32", "bf16"):
        return stored.double().numpy()
    if kv in ("int4", "fp4"):
        return kv4ref.decode(stored.numpy(), scale.numpy(), kv)
    v = stored.view(torch.int8 if kv == "int8" else torch.float8_e4m3fn)
    return (v.float().double() * scale.double().unsqueeze(-1)).numpy()


def attend(q, k, v, seen, kscale, vscale, kv):
    """Attention of q over the rows `seen` of k and v (64 bits), and how far a float evaluation with weights in two bf16
    halves (F32 caches: in float) may be from it.

    Scores: 64 products, exact for bf16 q and codes, a float rounding each for F32, summed in float in any order: 70
    roundings of 2^-24 of the sum of magnitudes, in which an INT4 code counts 15 + 8 (the operand adds 8, and -8 times
    the sum of q starts the sum); two roundings of the scale's product; the exponent's difference rounds once more.  A
    weight is exp2 of that (2^-22 for the instruction); over BF16 rows it is cut to two bf16 halves (2^-14), over codes its
    product with the row's scale, with room for a float16 of it (2^-11).  Sums: a rounding for each 32 rows of a product,
    the joins of waves and segments, the total's division; then half a step of the output."""
    n = len(seen)
    if n == 0:
        return np.zeros(HS), np.full(HS, 2.0 ** -126)
    k, v = k[seen], v[seen]
    s = k @ q / 8.0
    w = np.exp(s - s.max())
    w /= w.sum()
    ref = w @ v
    more = 23.0 if kv == "int4" else 0.0
    mag = (np.abs(k) @ np.abs(q)).max() + more * np.abs(q).sum() * (kscale[seen].max() if more else 0.0)
    es = 2 * 74 * 2.0 ** -24 * mag * 0.125 * LOG2E
    rel_w = {"f32": 0.0, "bf16": 2.0 ** -14}.get(kv, 2.0 ** -11) + 2.0 ** -21 + 2 * math.log(2) * es
    size = np.abs(v).max() + more * (vscale[seen].max() if more else 0.0)
    steps = (n / 4 + 24) * 2.0 ** -24 if kv == "f32" else (n / 32 + 24) * 2.0 ** -24
    half = HALF_STEP["f32" if kv == "f32" else "bf16"]
    return ref, half * np.abs(ref) + 2 * rel_w * (w @ np.abs(v)) + 2 * steps * size + 2.0 ** -126


# ------------------------------------------------------------------------------------
# The walk.
# ------------------------------------------------------------------------------------
def _mass(x):
    return float(x) if np.isfinite(x) and x > 0 else 0.0


def walk(p, tokens, parents, u, draw, t0, n):
    """-> accepted and drawn tokens, path (indices)."""
    V = p.shape[1]
    at, path, out = 0, [0], []
    n = min(n, 256)
    while True:
        upto, tried, nxt = 0.0, [], -1
        for c in range(1, n):
            if int(parents[t0 + c]) != at or at >= c:
                continue
            x = int(tokens[t0 + c])
            if x in tried:
                continue
            tried.append(x)
            upto += _mass(p[t0 + at, x]) if 0 <= x < V else 0.0
            if float(u[t0 + at]) < upto:
                nxt = c
                break
        if nxt < 0:
            break
        at = nxt
        path.append(at)
        out.append(int(tokens[t0 + at]))
    w = np.array([_mass(x) for x in p[t0 + at]])
    rest = w.copy()
    for x in tried:
        if 0 <= x < V:
            rest[x] = 0.0
    if rest.sum() > 0:
        w = rest
    if w.sum() > 0:
        c = np.cumsum(w)
        hit = int(np.searchsorted(c, float(draw) * c[-1], side="right"))
        out.append(min(hit, int(np.nonzero(w)[0].max())))
    return out, path


# ------------------------------------------------------------------------------------
# Rules on logits.
# ------------------------------------------------------------------------------------
def rules(x, held, made, r, f, pr, bias, allowed):
    """One row in 64 bits, and how far a float evaluation may be from it.  held, made: ids (with repeats); bias: {id: value};
    allowed: bool [V] or None.

    A quotient or product, a product and a sum, a difference, a sum: five roundings of 2^-24 of magnitudes that add up."""
    V = len(x)
    x = x.astype(np.float64).copy()
    count = np.bincount([t for t in made if 0 <= t < V], minlength=V).astype(np.float64)
    here = np.zeros(V, dtype=bool)
    here[[t for t in held if 0 <= t < V]] = True
    with np.errstate(invalid="ignore"):
        x = np.where(here, np.where(x > 0, x / r, x * r), x)
        size = np.abs(x) + abs(f) * count + abs(pr) * (count > 0)      # (f may be negative, its product's rounding is not)
        x = x - (f * count + pr * (count > 0))
        for t, b in bias.items():
            if 0 <= t < V:
                size[t] += abs(b)
                x[t] += b
    err = np.where(here | np.isin(np.arange(V), list(bias)), 5 * 2.0 ** -24 * size, 0.0)
    if allowed is not None:
        x[~allowed] = -np.inf
        err[~allowed] = 0.0
    return x, err


def softmax(x, err, T):
    """Probabilities of a row in 64 bits, and a float evaluation's distance: a weight's exponent has the logit's error
    and the maximum's, rounds at the difference, the factor (a quotient), the product (4 of 2^-24 of it), the
    instruction 2^-22; the sum has a rounding a token of a thread (70) and the join's 26, the quotient two more."""
    top = x.max()
    if top == -np.inf:
        return np.zeros_like(x), np.zeros_like(x)
    if not T > 0:
        p = np.zeros_like(x)
        p[int(np.argmax(x))] = 1.0
        return p, np.zeros_like(x)
    with np.errstate(invalid="ignore"):
        e = (x - top) / T
        p = np.exp(e)
        p /= p.sum()
        own = 2 * (err + err[np.isfinite(x)].max()) / T + 4 * 2.0 ** -24 * np.where(np.isfinite(e), np.abs(e), 0.0) + 2.0 ** -21
    rel = own + (p * own).sum() + 100 * 2.0 ** -24
    return p, 2 * rel * p + 2.0 ** -120


# ------------------------------------------------------------------------------------
# 4-bit weights.
# ------------------------------------------------------------------------------------
def w4_codes(W, group, kind):
    """W [M][K] float32 -> nibbles [M][K], scales [M][K/group] (float32 holding bf16), as w4_quantize defines them."""
    M, K = W.shape
    g = W.reshape(M, K // group, group).astype(np.float32)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        amax = np.fmax.reduce(np.abs(g), axis=-1, initial=np.float32(0))
        scale = bf16((amax / np.float32(7 if kind == "int4" else 6)).astype(np.float32))
        y = np.where(scale[..., None] > 0, g / scale[..., None], np.float32(0)).astype(np.float32)
    y = np.where(np.isnan(y), np.float32(0), y).reshape(M, K)
    if kind == "int4":
        return (np.clip(np.rint(y), -7, 7) + 8).astype(np.uint8), scale
    a = np.abs(y)
    mag = np.zeros(a.shape, dtype=np.uint8)
    for i, m in enumerate((kv4ref.FP4[1:] + kv4ref.FP4[:-1]) / 2):
        mag += (a > m) if i % 2 == 0 else (a >= m)
    return mag | (np.signbit(y).astype(np.uint8) << 3), scale


def w4_values(nib, scale, kind):
    code = nib.astype(np.float64) - 8 if kind == "int4" else np.where(nib & 8, -1.0, 1.0) * kv4ref.FP4[nib & 7]
    return code * np.repeat(scale.astype(np.float64), nib.shape[1] // scale.shape[1], axis=1)


def gelu(y):
    return 0.5 * y * (1 + np.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))


def w4_layer(nib, scale, x, bias, kind):
    """x W^T + bias in 64 bits and a float evaluation's distance: products are exact; a group's sum, a rounding each 8
    products and 4 for -8 times x's (INT4: magnitudes of 15 + 8 a code); its scale's product, the sum over groups, waves
    and bias."""
    W = w4_values(nib, scale, kind)
    ref = x @ W.T + bias
    top = np.repeat(scale.astype(np.float64), nib.shape[1] // scale.shape[1], axis=1)
    mag = np.abs(x) @ ((23.0 * top) if kind == "int4" else np.abs(W)).T
    steps = 32 + nib.shape[1] / 32 + 12
    return ref, steps * 2.0 ** -24 * (mag + np.abs(bias))
