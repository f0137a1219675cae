"""The cache in pages on the GPU: append with rotation, attention of one query per sequence, attention of ragged new tokens, and a
run of them together, against NumPy in 64 bits (tests/paged_ref.py, which derives the bounds)."""
import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


class OnDevice:
    """A Batch's arrays on the device, through the public calls."""

    def __init__(self, ex, b, max_kv_len=None):
        self.b = b
        self.table, self.kv_len = ex.to_device(b.table), ex.to_device(b.kv_len)
        self.cu = None if b.cu is None else ex.to_device(b.cu)
        self.pool = ex.paged_kv(b.n_pages, b.page, b.n_kv, b.hd)
        self.k, self.v = self.pool.pages()
        self.k.upload(b.k.view(np.uint16)), self.v.upload(b.v.view(np.uint16))
        self.seqs = ex.paged_seqs(self.table, self.kv_len, b.n_seq, b.max_blocks, self.cu, int(max(b.kv_len)) if max_kv_len is None else max_kv_len)

    def pages(self):
        shape = self.b.k.shape
        return self.k.download(np.uint16).reshape(shape), self.v.download(np.uint16).reshape(shape)


# ---------------------------------------------------------------------------------------------------------------- append


@pytest.mark.parametrize("rope", ["interleaved", "half", "none"])
@pytest.mark.parametrize("hd,page,n_kv,n_heads,kv_len,new", [
    (128, 16, 2, 4, [5, 0, 16, 33], [5, 0, 1, 17]),
    (64, 32, 3, 3, [1, 32, 70], [1, 32, 3]),
    (64, 16, 1, 5, [40], [40]),
    (128, 64, 4, 4, [64, 65, 1, 2], None),
    (64, 16, 2, 2, [7, 0, 19], None),
    (128, 1024, 1, 8, [131071, 9], [2, 9]),
])
def test_append_turns_and_stores(ex, rope, hd, page, n_kv, n_heads, kv_len, new):
    print("append", rope, hd, page, n_kv, n_heads, kv_len, new, flush=True)
    rng = np.random.default_rng(hash((hd, page, n_kv)) % 1000)
    b = ref.Batch(rng, kv_len, page, n_kv, hd, new)
    d = OnDevice(ex, b)
    n_tok = b.n_seq if new is None else sum(new)
    # keys and values are slices of one row that holds both, queries have a gap behind them
    row, rowkv = n_heads * hd, n_kv * hd
    kvrow = rng.standard_normal((n_tok, 2 * rowkv + 8)).astype(np.float32)
    q = rng.standard_normal((n_tok, row + 4)).astype(np.float32)
    dkv, dq = ex.to_device(kvrow), ex.to_device(q)
    dv = ex.borrow(dkv.ptr.value + 4 * rowkv, dkv.nbytes - 4 * rowkv)
    dout = ex.to_device(np.full((n_tok, row + 12), 7.0, dtype=np.float32))
    theta = 500000.0
    ex.paged_append_dev(d.pool, d.seqs, dkv, dv, n_tok, q=dq, q_out=dout, n_heads=n_heads, rope=rope, theta=theta, k_ld=2 * rowkv + 8, v_ld=2 * rowkv + 8,
                        q_ld=row + 4, q_out_ld=row + 12)
    got_q = dout.download(np.float32).reshape(n_tok, row + 12)
    got_k, got_v = d.pages()
    want_k, want_v = b.k.view(np.uint16).copy(), b.v.view(np.uint16).copy()
    assert (got_q[:, row:] == 7.0).all()
    told = set()
    for t, s, pos in b.places():
        if pos < 0:
            continue
        told.add(t)
        x = q[t, :row].astype(np.float64).reshape(n_heads, hd)
        k = kvrow[t, :rowkv].astype(np.float64).reshape(n_kv, hd)
        if rope == "none":
            assert np.array_equal(got_q[t, :row], q[t, :row])
            kt, mag = k, np.zeros_like(k)
        else:
            y, m = ref.turn(x, pos, rope, theta)
            assert (np.abs(got_q[t, :row].reshape(n_heads, hd) - y) <= ref.TURN * m).all()
            kt, mag = ref.turn(k, pos, rope, theta)
        pg, sl = b.table[s, pos // page], pos % page
        got = got_k[pg, :, sl].view(np.float16).astype(np.float64)
        assert (np.abs(got - kt) <= ref.U16 * (np.abs(kt) + ref.TURN * mag) + ref.TURN * mag + 2.0 ** -25).all()
        v = kvrow[t, rowkv:2 * rowkv].reshape(n_kv, hd).astype(np.float16)
        assert np.array_equal(got_v[pg, :, sl], v.view(np.uint16))          # rounded to nearest even, bit for bit
        want_k[pg, :, sl], want_v[pg, :, sl] = got_k[pg, :, sl], got_v[pg, :, sl]
    assert np.array_equal(got_k, want_k) and np.array_equal(got_v, want_v)      # every other slot as it was
    for t in range(n_tok):
        if t not in told:
            assert (got_q[t] == 7.0).all()                                       # an idle sequence's row


def test_append_in_place_equals_append_beside(ex):
    rng = np.random.default_rng(5)
    b = ref.Batch(rng, [20, 31], 16, 2, 128, [4, 31])
    x = rng.standard_normal((35, 4 * 128)).astype(np.float32)
    kv = ex.to_device(rng.standard_normal((35, 2 * 128)).astype(np.float32))
    got = []
    for in_place in (False, True):
        d = OnDevice(ex, b)
        dq = ex.to_device(x)
        dout = dq if in_place else ex.buffer(x.nbytes)
        ex.paged_append_dev(d.pool, d.seqs, kv, kv, 35, q=dq, q_out=dout, n_heads=4)
        got.append((dout.download(np.float32), *d.pages()))
    assert all(np.array_equal(a, c) for a, c in zip(*got))
    d = OnDevice(ex, b)                          # and without queries at all
    ex.paged_append_dev(d.pool, d.seqs, kv, kv, 35)
    assert all(np.array_equal(a, c) for a, c in zip(d.pages(), got[0][1:]))


def test_append_leaves_what_the_batch_does_not_own(ex):
    """Rows before the first and behind the last sequence, pages that are not the pool's, positions beyond the table."""
    rng = np.random.default_rng(6)
    b = ref.Batch(rng, [18, 40, 33], 16, 1, 64, [2, 8, 33], extra_blocks=0)
    b.cu = np.array([3, 5, 13, 46], dtype=np.int32)              # rows 0..2 and 46.. belong to nobody
    b.table[1, 2] = b.n_pages                                     # positions 32.. of sequence 1
    b.table[2, 0], b.table[2, 1] = -7, 2 ** 31 - 1
    b.kv_len[0] = 16 * b.max_blocks + 1                           # its last token lies beyond the table
    d = OnDevice(ex, b)
    q = rng.standard_normal((50, 64)).astype(np.float32)
    kv = rng.standard_normal((50, 64)).astype(np.float32)
    dout = ex.to_device(np.full((50, 64), 7.0, dtype=np.float32))
    dkv = ex.to_device(kv)
    ex.paged_append_dev(d.pool, d.seqs, dkv, dkv, 50, q=ex.to_device(q), q_out=dout, n_heads=1, rope="none")
    got_q, (got_k, got_v) = dout.download(np.float32).reshape(50, 64), d.pages()
    assert (got_q[:3] == 7).all() and (got_q[46:] == 7).all() and np.array_equal(got_q[3:46], q[3:46])
    want_k, want_v = b.k.copy(), b.v.copy()
    for s in range(3):
        for i in range(b.new[s]):
            t, pos = int(b.cu[s]) + i, int(b.kv_len[s]) - b.new[s] + i
            if pos // 16 < b.max_blocks and 0 <= b.table[s, pos // 16] < b.n_pages:
                want_k[b.table[s, pos // 16], 0, pos % 16] = want_v[b.table[s, pos // 16], 0, pos % 16] = kv[t].astype(np.float16)
    assert np.array_equal(got_k, want_k.view(np.uint16)) and np.array_equal(got_v, want_v.view(np.uint16))


# ------------------------------------------------------------------------------------------------------- decode attention


def check_decode(ex, rng, b, n_heads, max_kv_len=None, q_scale=1.0):
    d = OnDevice(ex, b, max_kv_len)
    row = n_heads * b.hd
    q = (rng.standard_normal((b.n_seq, row + 4)) * q_scale).astype(np.float32)
    dout = ex.to_device(np.full((b.n_seq + 1, row + 8), 7.0, dtype=np.float32))
    ex.paged_attn_decode_dev(d.pool, d.seqs, ex.to_device(q), n_heads, dout, q_ld=row + 4, out_ld=row + 8)
    got = dout.download(np.float32).reshape(b.n_seq + 1, row + 8)
    assert (got[:, row:] == 7.0).all() and (got[b.n_seq] == 7.0).all()
    group = n_heads // b.n_kv
    for s in range(b.n_seq):
        for h in range(n_heads):
            _, k, v = b.rows(s, h // group, int(b.kv_len[s]))
            want, bound = ref.attention(q[s, h * b.hd:(h + 1) * b.hd].astype(np.float64), k, v, b.hd ** -0.5)
            diff = np.abs(got[s, h * b.hd:(h + 1) * b.hd] - want)
            assert (diff <= bound).all(), (s, h, int(b.kv_len[s]), float((diff / bound).max()))
    return got


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_kv,n_heads,page,kv_len", [
    (1, 1, 16, [1, 2, 15, 16, 17, 31, 32, 33]),
    (2, 2, 32, [63, 64, 65, 0, 127, 128, 129]),
    (2, 8, 16, [0, 255, 256, 257, 300]),
    (1, 5, 64, [511, 1, 513]),
    (1, 8, 128, [640]),
    (2, 24, 16, [77, 1, 0]),
    (1, 16, 256, [257]),
    (1, 17, 16, [90]),
    (1, 40, 16, [35]),
    (3, 6, 16, [1030]),
])
def test_decode_attention(ex, hd, n_kv, n_heads, page, kv_len):
    print("decode", hd, n_kv, n_heads, page, kv_len, flush=True)
    rng = np.random.default_rng(hd + n_heads)
    # what is not the sequences' own is NaN: stale slots behind a sequence's end, pages of nobody
    b = ref.Batch(rng, kv_len, page, n_kv, hd, fill=np.nan)
    for s in range(b.n_seq):
        b.put(rng, s)
    check_decode(ex, rng, b, n_heads)


@pytest.mark.parametrize("hint", [0, 1, 100, 5000, 2 ** 30])
def test_decode_attention_whatever_the_launch_was_cut_for(ex, hint):
    rng = np.random.default_rng(9)
    b = ref.Batch(rng, [900, 3, 0, 1500], 32, 1, 64, fill=np.inf, extra_blocks=40)
    for s in range(4):
        b.put(rng, s)
    check_decode(ex, rng, b, 2, max_kv_len=hint)


def test_decode_attention_sharp_and_flat_scores(ex):
    """Scores of hundreds (one key takes all), of 1e-30, and queries of zeros (the mean of the values)."""
    rng = np.random.default_rng(10)
    for scale in (0.0, 1e-30, 100.0):
        b = ref.Batch(rng, [200, 33], 16, 1, 128)
        check_decode(ex, rng, b, 4, q_scale=scale)


def test_decode_attention_does_not_see_pages_outside_the_pool(ex):
    rng = np.random.default_rng(11)
    b = ref.Batch(rng, [100, 50, 20, 64], 16, 2, 64, extra_blocks=0)
    b.table[0, 1], b.table[0, 6], b.table[1, 0], b.table[2, :2] = -1, b.n_pages, 2 ** 31 - 1, -(2 ** 31)      # sequence 2 has nothing left
    b.kv_len[3] = 16 * b.max_blocks + 12345                                                                    # counts as the table's width
    b.table[3, :] = rng.permutation(b.n_pages)[:b.max_blocks]
    got = check_decode(ex, rng, b, 4)
    assert (got[2, :4 * 64] == 0).all()


def test_decode_attention_of_sequences_that_share_pages(ex):
    rng = np.random.default_rng(12)
    b = ref.Batch(rng, [80, 70, 75], 16, 1, 128)
    b.table[1, :4] = b.table[2, :4] = b.table[0, :4]
    check_decode(ex, rng, b, 4)


# ------------------------------------------------------------------------------------------------------ prefill attention


def check_prefill(ex, rng, b, n_heads, n_tok=None, q=None):
    d = OnDevice(ex, b)
    row = n_heads * b.hd
    n_tok = n_tok or int(b.cu[-1])
    if q is None:
        q = rng.standard_normal((n_tok, row + 4)).astype(np.float32)
    dout = ex.to_device(np.full((n_tok + 1, row + 8), 7.0, dtype=np.float32))
    ex.paged_attn_prefill_dev(d.pool, d.seqs, ex.to_device(q), n_tok, n_heads, dout, q_ld=q.shape[1], out_ld=row + 8)
    got = dout.download(np.float32).reshape(n_tok + 1, row + 8)
    assert (got[:, row:] == 7.0).all() and (got[n_tok] == 7.0).all()
    group = n_heads // b.n_kv
    told = np.zeros(n_tok, dtype=bool)
    for t, s, pos in b.places():
        told[t] = True
        for h in range(n_heads):
            _, k, v = b.rows(s, h // group, pos + 1)
            want, bound = ref.attention(q[t, h * b.hd:(h + 1) * b.hd].astype(np.float64), k, v, b.hd ** -0.5)
            diff = np.abs(got[t, h * b.hd:(h + 1) * b.hd] - want)
            assert (diff <= bound).all(), (t, s, pos, h, float((diff / bound).max()))
    assert (got[:n_tok][~told] == 7.0).all()
    return got[:n_tok, :row]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_kv,n_heads,page,new,prior", [
    (1, 1, 16, [1], [0]),
    (1, 1, 16, [33], [0]),
    (2, 2, 16, [31, 0, 32, 1], [0, 9, 1, 40]),
    (1, 4, 32, [65], [30]),
    (2, 8, 16, [3, 40], [63, 0]),
    (1, 5, 64, [27], [100]),
    (1, 12, 16, [11, 2], [5, 0]),
    (1, 1, 128, [129], [0]),
    (1, 2, 16, [130], [127]),
])
def test_prefill_attention(ex, hd, n_kv, n_heads, page, new, prior):
    print("prefill", hd, n_kv, n_heads, page, new, prior, flush=True)
    rng = np.random.default_rng(hd + n_heads + len(new))
    b = ref.Batch(rng, [a + c for a, c in zip(new, prior)], page, n_kv, hd, new, fill=np.nan)
    for s in range(b.n_seq):
        b.put(rng, s)
    check_prefill(ex, rng, b, n_heads)


def test_prefill_attention_leaves_rows_of_nobody_and_bad_pages_alone(ex):
    rng = np.random.default_rng(21)
    b = ref.Batch(rng, [40, 30, 5], 16, 1, 64, [20, 30, 8])       # sequence 2 says more new tokens than positions: its first rows see nothing
    b.cu = np.array([2, 22, 52, 60], dtype=np.int32)
    b.table[0, 1], b.table[1, 0] = -5, b.n_pages
    check_prefill(ex, rng, b, 2, n_tok=70)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_prefill_attention_earlier_rows_do_not_see_later_infinities(ex, bad):
    """A value that overflowed at a later position leaves the rows before it alone (0 times infinity never enters their sums)."""
    rng = np.random.default_rng(22)
    b = ref.Batch(rng, [50, 20], 16, 1, 128, [45, 20])
    pg = b.table[0, 30 // 16]
    b.v[pg, 0, 30 % 16, 5] = bad
    b.k[b.table[1, 0], 0, 9] = bad
    d = OnDevice(ex, b)
    q = rng.standard_normal((65, 2 * 128)).astype(np.float32)
    dout = ex.buffer(q.nbytes)
    ex.paged_attn_prefill_dev(d.pool, d.seqs, ex.to_device(q), 65, 2, dout)
    got = dout.download(np.float32).reshape(65, 2, 128)
    for t, s, pos in b.places():
        if (s == 0 and pos < 30) or (s == 1 and pos < 9):
            for h in range(2):
                _, k, v = b.rows(s, 0, pos + 1)
                want, bound = ref.attention(q[t, h * 128:(h + 1) * 128].astype(np.float64), k, v, 128 ** -0.5)
                assert (np.abs(got[t, h] - want) <= bound).all(), (t, s, pos)
        elif s == 0:
            assert not np.isfinite(got[t, :, 5]).any() and np.isfinite(np.delete(got[t], 5, axis=1)).all()


def test_prefill_in_chunks_equals_prefill_at_once(ex):
    """Rows seen by two cuts of the same prompt agree to the bound of both."""
    rng = np.random.default_rng(23)
    whole = ref.Batch(rng, [90], 16, 2, 64, [90])
    q = rng.standard_normal((90, 4 * 64 + 4)).astype(np.float32)
    a = check_prefill(ex, rng, whole, 4, q=q)
    whole.new, whole.cu = [23], np.array([0, 23], dtype=np.int32)
    c = check_prefill(ex, rng, whole, 4, q=q[67:].copy())
    assert np.abs(a[67:] - c).max() <= 1e-4


# ------------------------------------------------------------------------------------------------------ all of it together


def test_a_server_loop_of_all_operators(ex):
    """Three sequences: prompts appended and attended together, then steps in which a token per sequence is appended, attended and
    sampled from logits made of the attention's output, one sequence idle from the middle on; every step against 64 bits."""
    rng = np.random.default_rng(31)
    n_kv, n_heads, hd, page, vocab, n_seq = 2, 4, 64, 16, 300, 3
    row, rowkv = n_heads * hd, n_kv * hd
    prompts, steps, theta = [17, 1, 40], 6, 10000.0
    b = ref.Batch(rng, [p + steps for p in prompts], page, n_kv, hd, prompts, fill=np.nan)
    b.kv_len[:] = prompts
    d = OnDevice(ex, b, max_kv_len=max(prompts) + steps)
    head = ex.upload_qweight(0, vocab, row, (rng.standard_normal((vocab, row)) * 0.3).astype(np.float32))
    w64 = ex.dequant(head).astype(np.float64)
    emb = rng.standard_normal((vocab, row + 2 * rowkv)).astype(np.float32)       # a token's q, k, v
    K = [np.zeros((0, n_kv, hd)) for _ in prompts]
    V = [np.zeros((0, n_kv, hd)) for _ in prompts]

    def attend64(s, x, pos):
        x = x.astype(np.float64)
        K[s] = np.concatenate([K[s], ref.turn(x[row:row + rowkv].reshape(n_kv, hd), pos, "half", theta)[0].astype(np.float16).astype(np.float64)[None]])
        V[s] = np.concatenate([V[s], x[row + rowkv:].reshape(n_kv, hd).astype(np.float16).astype(np.float64)[None]])
        qt = ref.turn(x[:row].reshape(n_heads, hd), pos, "half", theta)[0]
        return np.concatenate([ref.attention(qt[h], K[s][:, h // 2], V[s][:, h // 2], hd ** -0.5)[0] for h in range(n_heads)])

    toks = [rng.integers(0, vocab, p) for p in prompts]
    x = emb[np.concatenate(toks)]
    dx = ex.to_device(x)
    ld = row + 2 * rowkv
    view = lambda buf, at: ex.borrow(buf.ptr.value + 4 * at, buf.nbytes - 4 * at)  # noqa: E731
    dq, dout = ex.buffer(4 * sum(prompts) * row), ex.buffer(4 * sum(prompts) * row)
    ex.paged_append_dev(d.pool, d.seqs, view(dx, row), view(dx, row + rowkv), sum(prompts), q=dx, q_out=dq, n_heads=n_heads, rope="half", theta=theta, k_ld=ld,
                        v_ld=ld, q_ld=ld)
    ex.paged_attn_prefill_dev(d.pool, d.seqs, dq, sum(prompts), n_heads, dout)
    got = dout.download(np.float32).reshape(-1, row)
    at = 0
    for s, p in enumerate(prompts):
        for i in range(p):
            want = attend64(s, x[at], i)
            assert np.abs(got[at] - want).max() <= 1e-3 * np.abs(want).max()     # a key's fp16 rounding may fall the other way
            at += 1
    cur = [int(t[-1]) for t in toks]
    step = ex.paged_seqs(d.table, d.kv_len, n_seq, b.max_blocks, None, max(prompts) + steps)
    dlog, dtok, dprob = ex.buffer(4 * n_seq * vocab), ex.buffer(4 * n_seq), ex.buffer(4 * n_seq)
    for i in range(steps):
        b.kv_len[:] = [p + min(i, 2) + 1 if s == 1 else p + i + 1 for s, p in enumerate(prompts)]
        if i == 3:
            b.kv_len[1] = 0                                     # sequence 1 is done: idle from here on
        if i >= 3:
            b.kv_len[1] = 0
        d.kv_len.upload(b.kv_len)
        x = emb[cur]
        dx = ex.to_device(x)
        ex.paged_append_dev(d.pool, step, view(dx, row), view(dx, row + rowkv), n_seq, q=dx, q_out=dq, n_heads=n_heads, rope="half", theta=theta, k_ld=ld, v_ld=ld,
                            q_ld=ld)
        ex.paged_attn_decode_dev(d.pool, step, dq, n_heads, dout)
        ex.qgemv_dev(head, dout, dlog, n_seq)
        u = rng.random(n_seq)
        ex.sample_dev(dlog, n_seq, vocab, ex.to_device(u), dtok, temperature=ex.to_device(np.float32([0.8, 1.0, 0.0])), top_k=ex.to_device(np.int32([20, 0, 0])),
                      top_p=ex.to_device(np.float32([0.9, 0.95, 1.0])), out_prob=dprob)
        out, logits = dout.download(np.float32, n_seq * row).reshape(n_seq, row), dlog.download(np.float32).reshape(n_seq, vocab)
        tok, prob = dtok.download(np.int32), dprob.download(np.float32)
        for s in range(n_seq):
            if b.kv_len[s] == 0:
                assert (out[s] == 0).all()
                continue
            want = attend64(s, x[s], int(b.kv_len[s]) - 1)
            assert np.abs(out[s] - want).max() <= 1e-3 * np.abs(want).max()
            assert np.abs(logits[s] - w64 @ out[s].astype(np.float64)).max() <= 1e-3 * np.abs(logits[s]).max() + 1e-3
            t, p, margin = ref.sample(logits[s], (0.8, 1.0, 0.0)[s], (20, 0, 0)[s], np.float32((0.9, 0.95, 1.0)[s]), 0.0, u[s])
            if s == 0:
                t, p, margin = ref.sample(logits[s], np.float32(0.8), 20, np.float32(0.9), 0.0, u[s])
            assert margin < 1e-9 or (tok[s] == t and abs(prob[s] - p) <= 1e-6 * p)
            cur[s] = int(tok[s])


# ------------------------------------------------------------------------------------------------------------- refusals


def test_paged_calls_refuse_what_they_cannot_do(ex):
    from rustorch_amd.errors import InvalidParameters, OutOfMemory, ShapeMismatch
    for args in ((0, 16, 1, 64), (4, 8, 1, 64), (4, 24, 1, 64), (4, 2048, 1, 64), (4, 16, 0, 64), (4, 16, 1, 96), (4, 16, 1025, 64), (2 ** 31, 16, 1, 64)):
        with pytest.raises(ShapeMismatch):
            ex.paged_kv(*args)
    with pytest.raises(OutOfMemory):
        ex.paged_kv(2 ** 31 - 1, 1024, 8, 128)
    buf = ex.buffer(4 * 16 * 64 * 2)
    with pytest.raises(ShapeMismatch):
        ex.wrap_paged_kv(buf, buf, 5, 16, 1, 64)
    with pytest.raises(InvalidParameters, match="aligned"):
        ex.wrap_paged_kv(ex.borrow(buf.ptr.value + 2, buf.nbytes - 2), buf, 3, 16, 1, 64)
    kv = ex.paged_kv(4, 16, 2, 64)
    ints, x = ex.to_device(np.zeros(64, dtype=np.int32)), ex.to_device(np.zeros(4096, dtype=np.float32))
    with pytest.raises(ShapeMismatch):
        ex.paged_seqs(ints, ints, 20, 4)
    with pytest.raises(ShapeMismatch):
        ex.paged_seqs(ints, ints, 8, 4, ex.buffer(32))
    seqs = ex.paged_seqs(ints, ints, 4, 4, ints)
    one = ex.paged_seqs(ints, ints, 4, 4)
    with pytest.raises(ShapeMismatch):
        ex.paged_append_dev(kv, one, x, x, 3)                                    # one token per sequence
    with pytest.raises(ShapeMismatch):
        ex.paged_append_dev(kv, seqs, x, x, 33)                                  # the buffers hold 32 rows
    with pytest.raises(ShapeMismatch):
        ex.paged_append_dev(kv, seqs, x, x, 4, k_ld=130)
    with pytest.raises(ShapeMismatch):
        ex.paged_append_dev(kv, seqs, x, x, 4, k_ld=64)
    with pytest.raises(InvalidParameters):
        ex.paged_append_dev(kv, seqs, x, x, 4, q=x)
    with pytest.raises(InvalidParameters):
        ex.paged_append_dev(kv, seqs, x, x, 4, q=x, q_out=x, n_heads=2, q_ld=128, q_out_ld=132)
    with pytest.raises(InvalidParameters):
        ex.paged_append_dev(kv, seqs, x, x, 4, rope="none of these")
    with pytest.raises(InvalidParameters):
        ex.paged_append_dev(kv, seqs, x, x, 4, theta=0.0)
    with pytest.raises(InvalidParameters, match="aligned"):
        ex.paged_append_dev(kv, seqs, ex.borrow(x.ptr.value + 4, 4096), x, 4)
    for heads in (0, 3, -2):
        with pytest.raises(ShapeMismatch):
            ex.paged_attn_decode_dev(kv, one, x, heads, x)
        with pytest.raises(ShapeMismatch):
            ex.paged_attn_prefill_dev(kv, seqs, x, 4, heads, x)
    with pytest.raises(InvalidParameters):
        ex.paged_attn_prefill_dev(kv, one, x, 4, 2, x)
    with pytest.raises(ShapeMismatch):
        ex.paged_attn_decode_dev(kv, one, x, 32, x)                              # the buffers hold two rows of 2048
    with pytest.raises(InvalidParameters):
        ex.paged_attn_decode_dev(kv, ex.paged_seqs(ints, ints, 4, 4, None, -1), x, 2, x)
    with pytest.raises(InvalidParameters, match="aligned"):
        ex.paged_attn_decode_dev(kv, one, ex.borrow(x.ptr.value + 8, 8192), 2, x)
    lib = ex.lib
    big = 1 << 40                                                                # refused by size before anything is looked at
    for n_tok in ((1 << 22) + 1, -1):
        assert lib.rt_hip_paged_append_dev(ex.ctx, kv.handle, ints.ptr, 4, ints.ptr, ints.ptr, 4, n_tok, x.ptr, big, x.ptr, big, None, 0, None, 0, 0, 0, 1.0) == 2
    assert lib.rt_hip_paged_attn_prefill_dev(ex.ctx, kv.handle, ints.ptr, 4, ints.ptr, ints.ptr, 4, 1 << 23, x.ptr, big, 2, x.ptr, big) == 2
    for n_seq, max_blocks in ((0, 4), (65536, 4), (4, 0), (4, (1 << 26) + 1)):
        assert lib.rt_hip_paged_attn_decode_dev(ex.ctx, kv.handle, ints.ptr, max_blocks, ints.ptr, n_seq, 0, x.ptr, 128, 2, x.ptr, 128) == 2
    assert lib.rt_hip_paged_attn_decode_dev(ex.ctx, kv.handle, ints.ptr, 4, ints.ptr, 65535, 0, x.ptr, 8192, 128, x.ptr, 8192) == 2
    ex.paged_append_dev(kv, seqs, x, x, 0)                                       # no tokens: nothing to do
    ex.paged_attn_prefill_dev(kv, seqs, x, 0, 2, x)
    assert lib.rt_hip_paged_kv_free(ex.ctx, None) == 0
    assert lib.rt_hip_paged_append_dev(None, None, None, 0, None, None, 0, 0, None, 0, None, 0, None, 0, None, 0, 0, 0, 0.0) == 1
    assert lib.rt_hip_paged_attn_decode_dev(ex.ctx, None, None, 0, None, 0, 0, None, 0, 0, None, 0) == 1
    assert lib.rt_hip_paged_attn_prefill_dev(ex.ctx, None, None, 0, None, None, 0, 0, None, 0, 0, None, 0) == 1
    ex.synchronize()


def test_prefill_attention_of_more_sequences_than_a_wave_has_lanes(ex):
    rng = np.random.default_rng(24)
    new = [int(x) for x in rng.integers(0, 4, 70)]
    b = ref.Batch(rng, [n + int(x) for n, x in zip(new, rng.integers(0, 20, 70))], 16, 1, 64, new)
    check_prefill(ex, rng, b, 3)
    check_decode(ex, rng, ref.Batch(rng, [int(x) for x in rng.integers(0, 400, 130)], 16, 1, 64), 1)


@pytest.mark.parametrize("group", [1, 4])
def test_prefill_attention_of_a_long_prompt(ex, group):
    """As many rows as the launch for full devices is taken for; every 37th row is looked at."""
    rng = np.random.default_rng(25)
    n, n_kv, hd = 1600, 8 * 4 // group, 64
    b = ref.Batch(rng, [n + 3], 64, n_kv, hd, [n])
    d = OnDevice(ex, b)
    q = rng.standard_normal((n, n_kv * group * hd)).astype(np.float32)
    dout = ex.buffer(q.nbytes)
    ex.paged_attn_prefill_dev(d.pool, d.seqs, ex.to_device(q), n, n_kv * group, dout)
    got = dout.download(np.float32).reshape(q.shape)
    for t in range(0, n, 37):
        h = (t * 7) % (n_kv * group)
        _, k, v = b.rows(0, h // group, 4 + t)
        want, bound = ref.attention(q[t, h * hd:(h + 1) * hd].astype(np.float64), k, v, hd ** -0.5)
        assert (np.abs(got[t, h * hd:(h + 1) * hd] - want) <= bound).all(), (t, h)


def test_two_executors_at_once(ex):
    """Two contexts, each with a stream and a workspace of its own, run split decode steps over one pool between one another."""
    from rustorch_amd.executor import HipKernelExecutor
    rng = np.random.default_rng(40)
    b = ref.Batch(rng, [3000, 1, 700], 16, 2, 64)
    d = OnDevice(ex, b)
    q = [rng.standard_normal((3, 4 * 64)).astype(np.float32) for _ in range(2)]
    with HipKernelExecutor(0) as other:
        outs = []
        for e, x in ((ex, q[0]), (other, q[1])):
            outs.append((e, e.to_device(x), [e.buffer(x.nbytes) for _ in range(4)]))
        pools = [e.wrap_paged_kv(d.k, d.v, b.n_pages, 16, 2, 64) for e, _, _ in outs]
        for i in range(4):
            for (e, dq, out), pool in zip(outs, pools):
                e.paged_attn_decode_dev(pool, d.seqs, dq, 4, out[i])
        for (e, _, out), x in zip(outs, q):
            got = [o.download(np.float32) for o in out]
            assert all(np.array_equal(got[0], g) for g in got)               # the same bits every time
            for s in range(3):
                for h in range(4):
                    _, k, v = b.rows(s, h // 2, int(b.kv_len[s]))
                    want, bound = ref.attention(x[s, h * 64:(h + 1) * 64].astype(np.float64), k, v, 1 / 8)
                    assert (np.abs(got[0].reshape(3, 4, 64)[s, h] - want) <= bound).all()
        for p in pools:
            p.free()
