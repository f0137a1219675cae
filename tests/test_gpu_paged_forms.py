"""Attention over pages in the launch forms that small cases do not take: prefill with 128 rows a workgroup (heads of 128, many rows), and
decode chunks of more pages than a wave holds table entries of; a sample of the heads against NumPy in 64 bits (tests/paged_ref.py)."""
from pathlib import Path

import numpy as np
import pytest

import paged_ref as ref
from test_gpu_paged import OnDevice
from test_gpu_paged_nonfinite import compare, definition, place

pytestmark = pytest.mark.gpu
SOURCE = Path(__file__).resolve().parents[1] / "rustorch_amd" / "csrc" / "rt_paged_attn.hip"


def takes_128_rows(n_tok, n_heads, n_kv, hd):
    """launch_paged_prefill's rule, and that it still is that rule."""
    assert "if ((long long)n_tok * a.group / 128 * p.n_kv >= 640) return run_prefill<128, 4, 1>(s, a);" in SOURCE.read_text()
    return hd == 128 and n_tok * (n_heads // n_kv) // 128 * n_kv >= 640


def run(ex, rng, b, n_heads, heads, q_scale=1.0, n_tok=None, check=None):
    n_tok = n_tok or int(b.cu[-1])
    assert takes_128_rows(n_tok, n_heads, b.n_kv, b.hd)
    d = OnDevice(ex, b)
    row = n_heads * b.hd
    q = rng.standard_normal((n_tok, row), dtype=np.float32) * np.float32(q_scale)
    dout = ex.to_device(np.full((n_tok + 1, row), 7.0, dtype=np.float32))
    ex.paged_attn_prefill_dev(d.pool, d.seqs, ex.to_device(q), n_tok, n_heads, dout)
    got = dout.download(np.float32).reshape(n_tok + 1, row)
    told = np.zeros(n_tok + 1, dtype=bool)
    for t, s, pos in b.places():
        told[t] = True
        for h in heads:
            at = slice(h * b.hd, (h + 1) * b.hd)
            _, k, v = b.rows(s, h // (n_heads // b.n_kv), pos + 1)
            want, bound = (check or (lambda q, k, v: ref.attention(q, k, v, b.hd ** -0.5)))(q[t, at].astype(np.float64), k, v)
            compare(got[t, at], want, bound, (t, s, pos, h))
    assert (got[~told] == 7.0).all()
    return got


def some(rng, n, m=5):
    return sorted({0, n - 1, *(int(h) for h in rng.integers(0, n, m))})


@pytest.mark.parametrize("n_kv,n_heads,page,new,prior,q_scale", [
    (640, 640, 16, [128], [0], 1.0),                                   # one tile of rows
    (320, 320, 16, [100, 0, 33, 1, 130], [0, 9, 40, 70, 3], 1.0),      # remainders, an empty sequence, one row
    (64, 256, 64, [321], [77], 1.0),                                   # four query heads' rows packed
    (64, 320, 32, [256], [31], 100.0),                                 # five, and scores of hundreds
])
def test_prefill_attention_of_128_rows_a_workgroup(ex, n_kv, n_heads, page, new, prior, q_scale):
    print("prefill, 128 rows", n_kv, n_heads, page, new, prior, q_scale, flush=True)
    rng = np.random.default_rng(n_heads + len(new))
    b = ref.Batch(rng, [a + c for a, c in zip(new, prior)], page, n_kv, 128, new, fill=np.nan)
    for s in range(b.n_seq):
        b.put(rng, s)
    run(ex, rng, b, n_heads, some(rng, n_heads), q_scale)


def test_prefill_attention_of_128_rows_and_more_sequences_than_lanes(ex):
    rng = np.random.default_rng(31)
    new = [int(x) for x in rng.integers(0, 8, 70)]
    new[33] = 140                                                      # tiles of one sequence among seventy
    b = ref.Batch(rng, [n + int(x) for n, x in zip(new, rng.integers(0, 30, 70))], 32, 320, 128, new)
    run(ex, rng, b, 320, some(rng, 320, 3))


def test_prefill_attention_of_128_rows_with_rows_of_nobody_and_bad_pages(ex):
    rng = np.random.default_rng(32)
    b = ref.Batch(rng, [140, 150, 20], 16, 320, 128, [120, 150, 25])   # sequence 2 says more new tokens than positions
    b.cu = np.array([2, 122, 272, 297], dtype=np.int32)
    b.table[0, 1], b.table[1, 0], b.table[1, 5] = -5, b.n_pages, 2 ** 31 - 1
    run(ex, rng, b, 320, some(rng, 320, 3), n_tok=300)


def test_prefill_attention_of_128_rows_with_values_and_keys_that_are_not_finite(ex):
    rng = np.random.default_rng(33)
    b = ref.Batch(rng, [290, 40], 16, 320, 128, [250, 40])
    heads = some(rng, 320, 2)
    for p, e, x in ((3, 1, np.inf), (50, 2, -np.inf), (200, 3, np.nan), (285, 4, np.inf), (120, 5, np.inf), (130, 5, -np.inf)):
        pg, sl = place(b, 0, p)
        b.v[pg, heads, sl, e] = x
    for s, p, x in ((0, 10, -np.inf), (1, 0, -np.inf), (0, 260, np.inf)):
        pg, sl = place(b, s, p)
        b.k[pg, heads, sl, 9] = x
    got = run(ex, rng, b, 320, heads, check=definition).reshape(-1, 320, 128)[:290, heads]
    assert np.isnan(got[:250]).any() and np.isinf(got[:250]).any() and np.isfinite(got[:250]).any()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_kv,n_heads,kv_len,hint", [(1, 2, [3000, 1025, 1024, 17], 1), (64, 64, [4500], 4500)])
def test_decode_attention_over_more_pages_than_lanes(ex, hd, n_kv, n_heads, kv_len, hint):
    """Chunks of more than 64 pages of 16: one chunk a sequence (the launch was cut for short ones), and four of a long one; pages
    outside the pool at both sides of a wave's window of table entries."""
    print("decode, many pages", hd, n_kv, n_heads, kv_len, hint, flush=True)
    rng = np.random.default_rng(hd)
    b = ref.Batch(rng, kv_len, 16, n_kv, hd)
    for p in (0, 63, 64, 127, 128, 187):
        if p % 2 == 0 or p == 63:
            b.table[0, p] = -1 if p % 3 else b.n_pages
    d = OnDevice(ex, b, hint)
    q = rng.standard_normal((b.n_seq, n_heads * hd), dtype=np.float32)
    dout = ex.buffer(q.nbytes)
    ex.paged_attn_decode_dev(d.pool, d.seqs, ex.to_device(q), n_heads, dout)
    got = dout.download(np.float32).reshape(q.shape)
    for s in range(b.n_seq):
        for h in some(rng, n_heads, 3):
            at = slice(h * hd, (h + 1) * hd)
            _, k, v = b.rows(s, h // (n_heads // n_kv), int(b.kv_len[s]))
            want, bound = ref.attention(q[s, at].astype(np.float64), k, v, hd ** -0.5)
            compare(got[s, at], want, bound, (s, h))
