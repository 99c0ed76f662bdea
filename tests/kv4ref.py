"""Plain restatements of the 4-bit cache types, the page bookkeeping and the draft verification
(numpy, 64 bits), and the error bounds that the tests hold the kernels to."""
import numpy as np

HS = 64
FP4 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
LIMIT = {"int4": np.float32(7), "fp4": np.float32(6)}
BIAS = {"int4": 24.0, "fp4": 0.0}       # what the INT4 operand adds to a code, and takes off again


def encode(x, kv):
    """Rows x [..., 64] (float32 holding bf16) -> packed bytes [..., 32], scales [...], as the types define."""
    x = np.asarray(x, dtype=np.float32)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        amax = np.fmax.reduce(np.abs(x), axis=-1, initial=np.float32(0))
        scale = (amax * (np.float32(1) / LIMIT[kv])).astype(np.float32)
        y = np.where(scale[..., None] > 0, x / scale[..., None], np.float32(0)).astype(np.float32)
    y = np.where(np.isnan(y), np.float32(0), y)
    if kv == "int4":
        nib = (np.clip(np.rint(y), -7, 7) + 8).astype(np.uint8)
    else:
        a = np.abs(y).astype(np.float64)
        mid = (FP4[1:] + FP4[:-1]) / 2
        mag = np.zeros(a.shape, dtype=np.uint8)
        for i, m in enumerate(mid):                   # ties to the even code
            mag += (a > m) if i % 2 == 0 else (a >= m)
        nib = mag | (np.signbit(y).astype(np.uint8) << 3)
    return (nib[..., 0::2] | (nib[..., 1::2] << 4)).astype(np.uint8), scale


def decode(packed, scale, kv):
    """Packed bytes and scales -> values in 64 bits."""
    nib = np.stack([packed & 15, packed >> 4], axis=-1).reshape(packed.shape[:-1] + (HS,))
    code = nib.astype(np.float64) - 8 if kv == "int4" else np.where(nib & 8, -1.0, 1.0) * FP4[nib & 7]
    return code * np.asarray(scale, dtype=np.float64)[..., None]


def attend(q, k, v, seen):
    """Attention of one query over the first `seen` rows, and sum of w |v| (64 bits)."""
    if seen <= 0:
        return np.zeros(HS), np.zeros(HS)
    s = k[:seen] @ q / 8.0
    w = np.exp(s - s.max())
    w /= w.sum()
    return w @ v[:seen], w @ np.abs(v[:seen])


def bound(ref, wv, q, kscale, vscale, kv, seen):
    """How far a float32 evaluation with bf16 output may be from attend().

    Scores: 64 products of bf16 q (exact) with codes of magnitude up to 7 + BIAS, summed in float in any
    order: 64 steps of 2^-24 of the sum of magnitudes, the BIAS's own sum likewise, two products more.
    A weight is exp2 of that (2^-22 for the instruction, and the difference's rounding of the same
    size as the score's), cut to two bf16 halves (2^-14).  Output: seen / 32 + 8 sums of float steps on
    terms of magnitude w (7 + BIAS) scale, two for the join of waves and segments; then half a step of
    bf16, 2^-8 of the value (2^-9 of a power of two's next), and of the smallest normal."""
    top = 7.0 + BIAS[kv]
    es = 0.0
    if seen > 0:
        es = 2 * 70 * 2.0 ** -24 * np.abs(q).sum() * top * np.abs(kscale[:seen]).max() * 0.125 * 1.4426950408889634
    rel_w = 2.0 ** -14 + 2.0 ** -22 + 2 * 0.6931471805599453 * es
    steps = (seen / 32 + 16) * 2.0 ** -24
    size = top * (np.abs(vscale[:seen]).max() if seen > 0 else 0.0)
    return 2.0 ** -8 * np.abs(ref) + 2 * rel_w * wv + 2 * steps * size + 2.0 ** -126


class Pool:
    """The page bookkeeping, request by request."""

    def __init__(self, num_pages, head=0, ring=None, count=None):
        self.P, self.head = num_pages, head
        self.ring = np.arange(num_pages, dtype=np.int32) if ring is None else np.array(ring, dtype=np.int32)
        self.count = num_pages if count is None else count

    def reserve(self, table, R, held, kept, fresh, max_tokens):
        """-> held_out, lens, token_start, slots, positions of one call (table and pool are updated)."""
        B, n = table.shape
        most = n * R
        up = lambda x: -(-x // R)                      # noqa: E731
        held_out, lens, start = np.array(held), np.array(kept), np.zeros(B + 1, dtype=np.int64)
        slots, positions, gone = [], [], []
        asked, took, tokens = 0, 0, 0
        for b in range(B):
            h, k, f = int(held[b]), int(kept[b]), int(fresh[b])
            sane = 0 <= k <= h <= most and f >= 0 and k + f <= most
            if not sane:
                start[b + 1] = tokens
                continue
            delta = up(k + f) - up(h)
            asked += max(delta, 0)
            tokens += f
            start[b + 1] = tokens
            ok = (delta <= 0 or asked <= self.count) and (f == 0 or tokens <= max_tokens)
            if ok:
                for i in range(delta):
                    table[b, up(h) + i] = self.ring[(self.head + took) % self.P]
                    took += 1
                gone += [table[b, i] for i in range(up(k + f), up(h))]
                held_out[b] = lens[b] = k + f
            for pos in range(k, k + f):
                page = table[b, pos // R] if ok else -1
                slots.append(int(page) * R + pos % R if 0 <= page < self.P else -1)
                positions.append(pos)
        for i, page in enumerate(gone):
            self.ring[(self.head + self.count + i) % self.P] = page
        self.head = (self.head + took) % self.P
        self.count += len(gone) - took
        return held_out, lens, start, np.array(slots[:max_tokens]), np.array(positions[:max_tokens])


def verify(p, q, drafts, u, start, V):
    """-> tokens (-2 where nothing is written), counts.  p, q float64 [rows, >= V]; q None: sure drafts."""
    tokens = np.full(len(u), -2, dtype=np.int64)
    counts = []

    def mass(w):
        w = np.array(w, dtype=np.float64)
        w[~(w > 0) | np.isinf(w)] = 0.0
        return w
    for b in range(len(start) - 1):
        t0, t1 = start[b], start[b + 1]
        n = t1 - t0
        if n == 0:
            counts.append(0)
            continue
        row = n - 1
        for i in range(n - 1):
            x, t = drafts[t0 + i], t0 + i
            if not (0 <= x < V and float(u[t]) * (1.0 if q is None else q[t, x]) < p[t, x]):
                row = i
                break
        w = np.array(p[t0 + row, :V])
        if row < n - 1:
            x = drafts[t0 + row]
            if q is not None:
                rest = mass(w - q[t0 + row, :V])
            else:
                rest = mass(w)
                if 0 <= x < V:
                    rest[x] = 0.0
            w = rest if rest.sum() > 0 else mass(w)
        else:
            w = mass(w)
        tokens[t0:t1] = -1
        tokens[t0:t0 + row] = drafts[t0:t0 + row]
        drawn = -1
        if w.sum() > 0:
            c = np.cumsum(w)
            over = np.nonzero((c > float(u[t1 - 1]) * c[-1]) & (w > 0))[0]
            drawn = over[0] if len(over) else np.nonzero(w)[0][-1]
            tokens[t0 + row] = drawn
        counts.append(row + (drawn >= 0))
    return tokens, np.array(counts)
