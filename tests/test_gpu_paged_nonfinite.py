"""Attention over pages where the cache holds infinities and NaN: what the definition leaves finite stays finite and right, what it
makes infinite or NaN comes out as that, in every form of the kernels, against NumPy in 64 bits (tests/paged_ref.py)."""
import numpy as np
import pytest

import paged_ref as ref
from test_gpu_paged import OnDevice

pytestmark = pytest.mark.gpu


def definition(q, k, v):
    """(out, bound) of one query, whose scores may be infinite or NaN: positions that score -inf weigh nothing (their values count
    as 0 times the value), a score of +inf or NaN makes the row NaN, and a value that is seen with a weight enters as it is."""
    n, hd = k.shape
    with np.errstate(all="ignore"):
        terms = np.where(q == 0, np.where(np.isfinite(k), 0.0, np.nan), k * q)
        s = np.where(np.isnan(terms).any(1), np.nan, terms.sum(1)) if n else np.zeros(0)
    if np.isnan(s).any() or (s == np.inf).any():
        return np.full(hd, np.nan), np.zeros(hd)
    on = s > -np.inf
    if not on.any():
        return np.where(np.isfinite(v).all(0), 0.0, np.nan), np.full(hd, 1e-30)
    finite = np.where(np.isfinite(v), v, 0.0)
    want, bound = ref.attention(q, k[on], finite[on], hd ** -0.5)
    bad = np.where(on[:, None], v, np.where(np.isfinite(v), 0.0, np.nan))          # 0 times what is not finite is NaN
    with np.errstate(all="ignore"):
        special = np.where(np.isfinite(bad), 0.0, bad).sum(0)                      # inf, -inf, or NaN, also of inf and -inf together
    return want + special, bound


def compare(got, want, bound, what):
    finite = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (what, "NaN where none belongs, or none where one does", got[np.isnan(got) != np.isnan(want)][:4], want[np.isnan(got) != np.isnan(want)][:4])
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)]), (what, "infinities")
    diff = np.abs(got[finite] - want[finite])
    assert (diff <= bound[finite]).all(), (what, float((diff / bound[finite]).max()))


def decode(ex, b, q, n_heads, max_kv_len=None):
    d = OnDevice(ex, b, max_kv_len)
    dout = ex.buffer(q.nbytes)
    ex.paged_attn_decode_dev(d.pool, d.seqs, ex.to_device(q), n_heads, dout)
    got = dout.download(np.float32).reshape(q.shape)
    for s in range(b.n_seq):
        for h in range(n_heads):
            at = slice(h * b.hd, (h + 1) * b.hd)
            _, k, v = b.rows(s, h // (n_heads // b.n_kv), int(b.kv_len[s]))
            compare(got[s, at], *definition(q[s, at].astype(np.float64), k, v), ("decode", s, h))
    return got


def prefill(ex, b, q, n_heads, rows=None, heads=None):
    d = OnDevice(ex, b)
    dout = ex.buffer(q.nbytes)
    ex.paged_attn_prefill_dev(d.pool, d.seqs, ex.to_device(q), len(q), n_heads, dout)
    got = dout.download(np.float32).reshape(q.shape)
    for t, s, pos in b.places():
        if rows is not None and t not in rows:
            continue
        for h in heads if heads is not None else range(n_heads):
            at = slice(h * b.hd, (h + 1) * b.hd)
            _, k, v = b.rows(s, h // (n_heads // b.n_kv), pos + 1)
            compare(got[t, at], *definition(q[t, at].astype(np.float64), k, v), ("prefill", t, s, pos, h))
    return got


def place(b, s, p):
    return b.table[s, p // b.page], p % b.page


def queries(rng, kind, rows, n):
    """Queries whose elements fill an f32, fit fp16 whole (nothing is left for a lower half), or lie many powers of two apart."""
    x = rng.standard_normal((rows, n))
    if kind == "halves":
        x = x.astype(np.float16)
    elif kind == "wide":
        x = x * 2.0 ** -rng.integers(0, 90, (rows, n)).astype(np.float64)
    x = x.astype(np.float32)
    assert (x != 0).all()
    return x


# ------------------------------------------------------------------------------------------------------------------ keys


@pytest.mark.parametrize("kind", ["f32", "halves", "wide"])
@pytest.mark.parametrize("hd", [64, 128])
def test_decode_attention_with_infinite_keys(ex, hd, kind):
    """An infinite element of a key scores -inf or +inf by the sign of the query's element: at -inf the position weighs nothing and
    the rest of the row is as ever."""
    print("decode, infinite keys", hd, kind, flush=True)
    rng = np.random.default_rng(hd)
    b = ref.Batch(rng, [40, 1, 700, 3], 16, 2, hd)
    for s, p, e, x in ((0, 7, 5, -np.inf), (0, 33, 5, -np.inf), (2, 0, 1, np.inf), (2, 650, 1, np.inf), (3, 1, 0, np.inf)):
        pg, sl = place(b, s, p)
        b.k[pg, :, sl, e] = x
    got = decode(ex, b, queries(rng, kind, 4, 8 * hd), 8)
    assert np.isfinite(got[1]).all() and np.isfinite(got).any(1).all() and np.isnan(got[[0, 2]]).any()


@pytest.mark.parametrize("kind", ["f32", "halves", "wide"])
@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_attention_with_infinite_keys(ex, hd, kind):
    print("prefill, infinite keys", hd, kind, flush=True)
    rng = np.random.default_rng(hd + 1)
    b = ref.Batch(rng, [70, 150], 16, 2, hd, [70, 40])
    for s, p, e, x in ((0, 3, 5, -np.inf), (0, 60, 6, np.inf), (1, 20, 2, np.inf), (1, 130, 2, -np.inf)):
        pg, sl = place(b, s, p)
        b.k[pg, :, sl, e] = x
    got = prefill(ex, b, queries(rng, kind, 110, 4 * hd), 4)
    assert np.isnan(got).any() and np.isfinite(got[10:70]).any()


def test_attention_over_keys_that_all_score_minus_infinity(ex):
    """Nothing weighs anything: zeros, as for a row that sees nothing."""
    rng = np.random.default_rng(3)
    b = ref.Batch(rng, [37, 300], 16, 1, 64, [5, 5])
    b.k[..., 11] = -np.inf
    q = np.abs(rng.standard_normal((10, 64))).astype(np.float32) + np.float32(0.01)
    assert (prefill(ex, b, q, 1) == 0).all()
    assert (decode(ex, b, q[:2].copy(), 1) == 0).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_prefill_attention_with_a_bad_first_key_and_a_later_bad_value(ex, bad):
    """A key that is no number at the first position makes every row NaN, also a row that is done again by itself because a value
    behind it is not finite; a score of -inf there weighs nothing, and 0 times an infinity is NaN also for a row of no weight."""
    rng = np.random.default_rng(4)
    b = ref.Batch(rng, [30, 30], 16, 1, 64, [30, 30])
    pg, sl = place(b, 0, 0)
    b.k[pg, 0, sl] = np.nan if np.isnan(bad) else b.k[pg, 0, sl]
    b.k[pg, 0, sl, 3] = bad
    pg, sl = place(b, 0, 20)
    b.v[pg, 0, sl, 9] = np.inf
    b.k[b.table[1, :2], 0, :, 5] = bad                           # sequence 1: every key
    b.v[b.table[1, 0], 0, 4, 2] = np.inf
    b.v[b.table[1, 1], 0, 4, 1] = np.nan
    got = prefill(ex, b, queries(rng, "f32", 60, 2 * 64), 2)
    assert np.isnan(got[:30]).any()


# ---------------------------------------------------------------------------------------------------------------- values


def bad_values(b, s, where):
    for p, e, x in where:
        pg, sl = place(b, s, p)
        b.v[pg, :, sl, e] = x


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_kv,n_heads,lens,new", [(2, 4, [200, 90], [40, 90]), (1, 1, [130], [130]), (1, 6, [333], [33])])
def test_prefill_attention_with_infinite_values_that_are_seen(ex, hd, n_kv, n_heads, lens, new):
    """A value of infinity that a row sees comes out as that infinity in its dim, both signs or a NaN as NaN, the other dims as ever:
    far before the rows, among them, and for the row whose only weight it is."""
    print("prefill, infinite values", hd, n_kv, n_heads, lens, new, flush=True)
    rng = np.random.default_rng(hd + n_heads)
    b = ref.Batch(rng, lens, 16, n_kv, hd, new)
    n = lens[0]
    bad_values(b, 0, [(0, 1, np.inf), (5, 2, -np.inf), (9, 3, np.nan), (n - 9, 4, np.inf), (n - 20, 4, -np.inf), (n - 7, 60, -np.inf), (n - 1, 7, np.nan)])
    got = prefill(ex, b, queries(rng, "f32", sum(new), n_heads * hd), n_heads)
    last = got[new[0] - 1].reshape(n_heads, hd)
    assert (last[:, 1] == np.inf).all() and (last[:, [2, 60]] == -np.inf).all() and np.isnan(last[:, [3, 4, 7]]).all() and np.isfinite(last[:, 8:60]).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_decode_attention_with_infinite_values(ex, hd):
    rng = np.random.default_rng(hd)
    b = ref.Batch(rng, [200, 1, 2000], 16, 2, hd)
    for s, n in ((0, 200), (1, 1), (2, 2000)):
        bad_values(b, s, [(0, 1, np.inf), (n // 2, 2, -np.inf), (n - 1, 3, np.nan), (0, 4, np.inf), (n - 1, 4, -np.inf if n > 1 else np.inf)])
    decode(ex, b, queries(rng, "f32", 3, 4 * hd), 4)


def test_prefill_attention_with_infinite_values_and_pages_outside_the_pool(ex):
    rng = np.random.default_rng(6)
    b = ref.Batch(rng, [120], 16, 1, 64, [70])
    b.k[b.table[0, 4]] = b.v[b.table[0, 4]] = np.nan
    bad_values(b, 0, [(3, 1, np.inf), (70, 2, np.nan), (110, 3, np.inf)])
    b.table[0, 4] = b.n_pages
    b.table[0, 2] = -1
    prefill(ex, b, queries(rng, "f32", 70, 2 * 64), 2)
