"""The paged operators and the sampling restated in NumPy, 64 bits, straight from their definitions; what the GPU tests compare with."""
import numpy as np

U32, U16 = 2.0 ** -24, 2.0 ** -11          # half a step of f32 and of fp16, relative


class Batch:
    """Host arrays of a batch of sequences over a pool: every sequence on pages of its own in a shuffled order, unused entries
    of the table out of range, pages filled with `fill` (stale contents)."""

    def __init__(self, rng, kv_len, page, n_kv, hd, new=None, fill=None, extra_blocks=1):
        self.kv_len = np.asarray(kv_len, dtype=np.int32)
        self.n_seq, self.page, self.n_kv, self.hd = len(kv_len), page, n_kv, hd
        blocks = [-(-max(0, int(x)) // page) for x in kv_len]
        self.max_blocks = max(1, max(blocks)) + extra_blocks
        self.n_pages = sum(blocks) + 2
        ids = rng.permutation(self.n_pages)
        self.table = np.full((self.n_seq, self.max_blocks), -1, dtype=np.int32)
        at = 0
        for s, b in enumerate(blocks):
            self.table[s, :b] = ids[at:at + b]
            at += b
        shape = (self.n_pages, n_kv, page, hd)
        if fill is None:
            self.k, self.v = rng.standard_normal(shape).astype(np.float16), rng.standard_normal(shape).astype(np.float16)
        else:
            self.k, self.v = np.full(shape, fill, dtype=np.float16), np.full(shape, fill, dtype=np.float16)
        self.new = None if new is None else [int(x) for x in new]
        self.cu = None if new is None else np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)

    def put(self, rng, s, scale=1.0):
        """Random keys and values for all positions of sequence s."""
        for p in range(int(self.kv_len[s])):
            pg, sl = self.table[s, p // self.page], p % self.page
            self.k[pg, :, sl] = (rng.standard_normal((self.n_kv, self.hd)) * scale).astype(np.float16)
            self.v[pg, :, sl] = rng.standard_normal((self.n_kv, self.hd)).astype(np.float16)

    def rows(self, s, kvh, n):
        """(positions, keys, values) of the first n positions of sequence s that lie on pages of the pool."""
        n = min(n, self.max_blocks * self.page)
        pos = np.array([p for p in range(n) if 0 <= self.table[s, p // self.page] < self.n_pages], dtype=np.int64)
        pg, sl = self.table[s, pos // self.page], pos % self.page
        return pos, self.k[pg, kvh, sl].astype(np.float64), self.v[pg, kvh, sl].astype(np.float64)

    def places(self):
        """(row, sequence, position) of every owned row of the new tokens."""
        if self.cu is None:
            return [(s, s, int(self.kv_len[s]) - 1) for s in range(self.n_seq)]
        return [(int(self.cu[s]) + i, s, int(self.kv_len[s]) - self.new[s] + i) for s in range(self.n_seq) for i in range(self.new[s])]


def turn(x, pos, style, theta):
    """x [heads, hd] in 64 bits turned by position `pos`, and for each element the sum of magnitudes its rounding errors scale with."""
    hd = x.shape[-1]
    i = np.arange(hd // 2)
    a = np.longdouble(pos) * np.longdouble(theta) ** (-2.0 * np.longdouble(1) * i / hd)
    c, s = np.cos(a).astype(np.float64), np.sin(a).astype(np.float64)
    first, second = (i, i + hd // 2) if style == "half" else (2 * i, 2 * i + 1)
    out, mag = np.empty_like(x), np.empty_like(x)
    p, q = x[..., first], x[..., second]
    out[..., first], out[..., second] = p * c - q * s, p * s + q * c
    mag[..., first] = mag[..., second] = np.abs(p) + np.abs(q)
    return out, mag


# A turned element: the angle, reduced in 64 bits, is rounded once to f32 (at most pi * 2^-24 off), sin and cos are off by at
# most 2 steps (4 * 2^-24) more, and two products and a sum round: (pi + 4 + 2) * 2^-24 of |p| + |q|.
TURN = 10 * U32


def attention(q, k, v, scale):
    """(out, bound) of one query over keys and values [n, hd] in 64 bits: the bound on an f32 implementation that accumulates in
    f32 in any order.  A score is off by at most d = (hd + 8) * 2^-24 * sum|q k| * scale (hd products summed, the operand split
    in two halves with 2^-22 left over, the scaling); a weight therefore by a factor exp(2 d) and 8 steps for the exponential;
    the sums over n positions add at most n + 32 steps each (numerator and denominator)."""
    n, hd = k.shape
    if n == 0:
        return np.zeros(hd), np.zeros(hd)
    s = (k @ q) * scale
    d = (hd + 8) * U32 * (np.abs(k) @ np.abs(q)).max() * scale
    w = np.exp(s - s.max())
    w /= w.sum()
    return w @ v, (2 * np.expm1(2 * d) + 2 * (n + 40) * U32) * (w @ np.abs(v)) + 1e-30


def sample(x, temperature, top_k, top_p, min_p, u):
    """(token, probability, margin): margin is how far (relative to the total) the nearest decision was from going the other way."""
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    top = x.max()
    if top == -np.inf:
        return -1, 0.0, 1.0
    best = int(np.flatnonzero(x == top)[0])
    if not temperature > 0 or top_k == 1:
        return best, 1.0, 1.0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    if top == np.inf:
        w = (x == top) * 1.0                      # beside an infinite logit everything finite weighs nothing
    else:
        w = np.where(x == -np.inf, 0.0, np.exp(np.where(x == -np.inf, 0.0, x - top) / temperature))
    margin = 1.0
    if 0 < top_p < 1:
        run = np.cumsum(w[order])
        cut = np.flatnonzero(run >= top_p * run[-1])[0]
        margin = min(margin, np.abs(run - top_p * run[-1]).min() / run[-1])
        order = order[:cut + 1]
    if min_p > 0:
        low = min(float(min_p), 1.0)
        keep = w[order] >= low
        off = np.abs(w[order] - low)
        margin = min(margin, off[off > 0].min() if (off > 0).any() else 1.0)
        order = order[keep]
    order = np.sort(order)
    order = order[w[order] > 0]
    run = np.cumsum(w[order])
    u = min(max(float(u), 0.0), 1.0)
    hit = np.flatnonzero(run > u * run[-1])
    at = int(hit[0]) if hit.size else run.size - 1
    if hit.size:
        margin = min(margin, np.abs(run - u * run[-1]).min() / run[-1]) if 0 < u < 1 else margin
    return int(order[at]), float(w[order[at]] / run[-1]), float(margin)
