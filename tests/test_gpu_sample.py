"""Sampling on the device against NumPy in 64 bits (tests/paged_ref.py) and against the host's sampling.py.  Token ids have to be
equal; a draw whose outcome hangs on less than 1e-11 of the total is not counted (64-bit sums in another order differ by that)."""
import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


def run(ex, x, temperature=None, top_k=None, top_p=None, min_p=None, u=0.5, ld=None):
    x = np.ascontiguousarray(x, dtype=np.float32)
    n, vocab = x.shape
    per_row = lambda v, t: None if v is None else ex.to_device(np.broadcast_to(np.asarray(v, dtype=t), (n,)))  # noqa: E731
    if ld:
        wide = np.full((n, ld), 1e30, dtype=np.float32)
        wide[:, :vocab] = x
    tok, prob = ex.to_device(np.full(n + 1, -5, dtype=np.int32)), ex.to_device(np.full(n + 1, 7, dtype=np.float32))
    ex.sample_dev(ex.to_device(wide if ld else x), n, vocab, per_row(u, np.float64), tok, temperature=per_row(temperature, np.float32), top_k=per_row(top_k, np.int32),
                  top_p=per_row(top_p, np.float32), min_p=per_row(min_p, np.float32), out_prob=prob, ld=ld)
    t, p = tok.download(np.int32), prob.download(np.float32)
    assert t[n] == -5 and p[n] == 7
    return t[:n], p[:n]


def check(ex, x, temperature=1.0, top_k=0, top_p=0.0, min_p=0.0, u=0.5, ld=None, borders=0):
    n = len(x)
    arr = lambda v, t: np.broadcast_to(np.asarray(v, dtype=t), (n,))  # noqa: E731
    T, k, p, m, uu = arr(temperature, np.float32), arr(top_k, np.int32), arr(top_p, np.float32), arr(min_p, np.float32), arr(u, np.float64)
    tok, prob = run(ex, x, T, k, p, m, uu, ld)
    near = 0
    for r in range(n):
        want, wp, margin = ref.sample(np.asarray(x[r], dtype=np.float32), float(T[r]), int(k[r]), float(p[r]), float(m[r]), float(uu[r]))
        if margin < 1e-11:
            near += 1
            continue
        # the probability: exp and the quotient in 64 bits, the total off by at most vocab * 2^-46 of it, one rounding to f32
        assert tok[r] == want and abs(prob[r] - wp) <= 2 * ref.U32 * wp, (r, tok[r], want, prob[r], wp, margin)
    assert near <= max(1, n // 10, borders)
    return tok


@pytest.mark.parametrize("vocab,rows,ld", [(1, 3, None), (2, 3, 5), (63, 4, 64), (1000, 5, None), (1025, 3, 2000), (32000, 3, None), (70001, 2, 70004)])
@pytest.mark.parametrize("temperature,top_k,top_p,min_p", [(1.0, 0, 0.0, 0.0), (0.7, 40, 0.95, 0.0), (1.3, 0, 0.9, 0.05), (1.0, 0, 0.0, 0.02), (0.0, 0, 0.0, 0.0),
                                                           (2.0, 7, 0.3, 0.5), (1.0, 2, 0.999, 0.0), (0.25, 700, 1.0, 0.0)])
def test_sampling(ex, vocab, rows, ld, temperature, top_k, top_p, min_p):
    print("sample", vocab, rows, ld, temperature, top_k, top_p, min_p, flush=True)
    rng = np.random.default_rng(vocab + top_k)
    x = rng.standard_normal((rows, vocab)) * 3
    check(ex, x, temperature, top_k, top_p, min_p, rng.random(rows), ld)


def test_rows_bring_their_own_settings(ex):
    rng = np.random.default_rng(3)
    n = 40
    x = rng.standard_normal((n, 501)) * 2
    check(ex, x, rng.choice([0.0, 0.5, 1.0, 4.0], n), rng.choice([-1, 0, 1, 3, 500, 501, 502, 2 ** 31 - 1], n), rng.choice([-1.0, 0.0, 0.2, 0.8, 1.0, 2.0], n),
          rng.choice([-1.0, 0.0, 0.1, 0.9, 1.0], n), rng.random(n))


def test_equal_logits_go_by_index(ex):
    n = 64
    u = (np.arange(n) + 0.5) / n
    flat = np.zeros((n, 100))
    assert check(ex, flat, 1.0, u=u).max() == 99
    assert check(ex, flat, 1.0, top_k=10, u=u).max() == 9                     # the first ten of a hundred equals
    assert check(ex, flat, 1.0, top_p=0.255, u=u).max() == 25                # 26 of them reach 25.5 %
    assert check(ex, flat, 1.0, top_k=40, top_p=0.255, u=u).max() == 10      # 11 of 40
    step = np.repeat(np.arange(5), 20)[None].repeat(n, 0) * 1.0              # ties at every level, the largest last
    step[:, ::2] = -step[:, ::2] * 0.0 + step[:, ::2]
    check(ex, step, 1.0, top_k=33, u=u)
    check(ex, step, 1.0, top_p=0.8, u=u)
    check(ex, step, 1.0, min_p=float(np.exp(-1.5)), u=u)
    zeros = np.where(np.arange(100) % 2, 0.0, -0.0)[None].repeat(4, 0)       # -0 and +0 are one value
    assert (check(ex, zeros, 0.0, u=0.9) == 0).all()
    assert check(ex, zeros, 1.0, top_k=3, u=[0.0, 0.4, 0.7, 0.99]).tolist() == [0, 1, 2, 2]


@pytest.mark.parametrize("pad", [0, 33000])
def test_infinities_and_nans(ex, pad):
    inf, nan = np.inf, np.nan
    rows = np.array([[0.0, -inf, 1.0, -inf, 2.0], [-inf, -inf, -inf, -inf, -inf], [nan, nan, nan, nan, nan], [nan, 1.0, nan, 2.0, -inf], [inf, 1.0, inf, 2.0, nan],
                     [-3.4e38, 3.4e38, 0.0, 1.0, -inf]])
    rows = np.pad(rows, ((0, 0), (0, pad)), constant_values=-inf)
    for u in (0.0, 0.3, 0.6, 0.999999):
        for kw in (dict(), dict(top_k=2), dict(top_p=0.5), dict(min_p=0.3), dict(temperature=0.0), dict(top_k=4, top_p=0.9, min_p=0.01), dict(temperature=1e30),
                   dict(temperature=1e-30), dict(temperature=inf)):
            check(ex, rows, u=u, **kw)
    tok, prob = run(ex, rows, u=0.5)
    assert tok[1] == tok[2] == -1 and prob[1] == prob[2] == 0


def test_edges_of_the_random_number_and_of_the_settings(ex):
    rng = np.random.default_rng(8)
    x = rng.standard_normal((6, 300))
    kept = np.sort(np.argsort(-x, axis=1, kind="stable")[:, :7], axis=1)
    tok, _ = run(ex, x, 1.0, 7, None, None, [0.0, 1.0 - 2.0 ** -53, 1.0, 7.0, -3.0, np.nan])
    assert tok.tolist() == [kept[0][0], kept[1][-1], kept[2][-1], kept[3][-1], kept[4][0], kept[5][0]]
    greedy = x.argmax(1)
    for t in (0.0, -1.0, np.nan):                              # a temperature that means nothing is the greedy pick
        assert (run(ex, x, t)[0] == greedy).all()
    assert (run(ex, x, 1.0, 1, u=0.99)[0] == greedy).all() and (run(ex, x, 1.0, None, None, 5.0, 0.99)[0] == greedy).all()
    a = run(ex, x, u=[0.1, 0.2, 0.3, 0.4, 0.5, 0.6])          # settings left out are off
    for kw in (dict(top_k=0), dict(top_p=np.nan), dict(min_p=np.nan), dict(top_p=1.0, top_k=300)):
        c = run(ex, x, 1.0, u=[0.1, 0.2, 0.3, 0.4, 0.5, 0.6], **kw)
        assert np.array_equal(a[0], c[0]) and np.array_equal(a[1], c[1])


def test_draws_follow_the_probabilities(ex):
    """Evenly spread random numbers hit every token as often as its probability says, to one draw on either side of its range."""
    rng = np.random.default_rng(9)
    n = 2000
    x = rng.standard_normal(50)
    p = np.exp(x / 0.8)
    p /= p.sum()
    tok, prob = run(ex, x[None].repeat(n, 0), 0.8, u=(np.arange(n) + 0.5) / n)
    assert (np.abs(np.bincount(tok, minlength=50) - n * p) <= 1.0 + 1e-4).all()
    assert np.allclose(prob, p[tok], rtol=1e-6)


def test_equals_the_host_sampler(ex):
    """The same random numbers through sampling.py's sample_token (64-bit probabilities) give the same tokens."""
    from rustorch_amd.sampling import SamplingConfig, sample_token

    class Given:
        def __init__(self, u):
            self.u = u

        def random(self):
            return self.u

    rng = np.random.default_rng(10)
    x = (rng.standard_normal((30, 800)) * 2).astype(np.float32)
    u = rng.random(30)
    for t, k, p in ((1.0, None, None), (0.5, 20, None), (1.0, None, 0.75), (2.0, 100, 0.5)):
        got, _ = run(ex, x, t, k, p, None, u)
        assert got.tolist() == [sample_token(x[r], SamplingConfig(t, k, p), rng=Given(u[r])) for r in range(30)]


def test_sampling_refuses_what_it_cannot_do(ex):
    from rustorch_amd.errors import ShapeMismatch
    x, u, t = ex.to_device(np.zeros(100, dtype=np.float32)), ex.to_device(np.zeros(4)), ex.to_device(np.zeros(4, dtype=np.int32))
    for rows, vocab, ld in ((4, 30, None), (4, 0, None), (-1, 10, None), (4, 20, 10), (1, (1 << 20) + 1, None), (65536, 0, 0)):
        with pytest.raises(ShapeMismatch):
            ex.sample_dev(x, rows, vocab, u, t, ld=ld)
    for kw in (dict(u=ex.buffer(24)), dict(out_token=ex.buffer(12)), dict(temperature=ex.buffer(12)), dict(top_k=ex.buffer(12)), dict(top_p=ex.buffer(12)),
               dict(min_p=ex.buffer(12)), dict(out_prob=ex.buffer(12))):
        with pytest.raises(ShapeMismatch):
            ex.sample_dev(x, 4, 25, **{**dict(u=u, out_token=t), **kw})
    ex.sample_dev(x, 0, 25, u, t)
    assert ex.lib.rt_hip_sample_dev(None, None, 0, 0, 0, None, None, None, None, None, None, None) == 1
    assert ex.lib.rt_hip_sample_dev(ex.ctx, None, 25, 4, 25, None, None, None, None, u.ptr, t.ptr, None) == 1
    assert ex.lib.rt_hip_sample_dev(ex.ctx, x.ptr, 25, 4, 25, None, None, None, None, None, t.ptr, None) == 1
    ex.synchronize()


@pytest.mark.parametrize("pad", [0, 40000])          # tokens that cannot be drawn behind the row's: one launch, and four
def test_thousands_of_equal_or_coarse_logits(ex, pad):
    """More tokens at one value than the device sorts, and logits on the grid that a 16-bit output leaves."""
    rng = np.random.default_rng(11)
    x = np.zeros((6, 5000))
    x[:, 4000:] = -0.5
    x[3:, 777] = 1.0
    x = np.pad(x, ((0, 0), (0, pad)), constant_values=-np.inf)
    u = [0.0, 0.3, 0.99, 0.01, 0.5, 0.9]
    for kw in (dict(), dict(top_k=2500), dict(top_k=4500, top_p=0.6), dict(top_p=0.99), dict(min_p=0.5), dict(top_k=3, min_p=0.9), dict(top_k=2500, temperature=1e-3)):
        # of 2500 equal tokens 0.3 and 0.99 end exactly behind the 750th and the 2475th: those two rows may go either way
        check(ex, x, u=u, borders=2, **kw)
    coarse = (rng.standard_normal((4, 20000)) * 2).astype(np.float32)
    coarse = (coarse.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
    coarse = np.pad(coarse, ((0, 0), (0, pad)), constant_values=-np.inf)
    for kw in (dict(), dict(top_k=50), dict(top_k=3000, top_p=0.7), dict(top_p=0.9), dict(top_p=0.5, min_p=0.2), dict(temperature=8.0, top_p=0.95), dict(temperature=0.05, top_p=0.95)):
        check(ex, coarse, u=rng.random(4), **kw)


def test_rows_of_a_large_vocabulary_with_their_own_settings(ex):
    rng = np.random.default_rng(13)
    x = rng.standard_normal((24, 50000)) * 2.5
    check(ex, x, rng.choice([0.0, 0.5, 1.0, 3.0], 24), rng.choice([0, 1, 3, 900, 1024, 1025, 4000, 49999], 24), rng.choice([0.0, 0.3, 0.9, 0.9999], 24),
          rng.choice([0.0, 0.01, 0.5], 24), rng.random(24))


def test_more_rows_than_one_launch_takes(ex):
    rng = np.random.default_rng(12)
    big = np.full((1100, 33000), -np.inf, dtype=np.float32)      # more rows than the four launches take at a time
    big[:, ::1100] = rng.standard_normal((1100, 30))
    check(ex, big, 0.9, rng.integers(0, 12, 1100), rng.choice([0.0, 0.7], 1100), rng.choice([0.0, 0.1], 1100), rng.random(1100))
    x = rng.standard_normal((1500, 40))
    check(ex, x, 0.9, rng.integers(0, 12, 1500), rng.choice([0.0, 0.7], 1500), rng.choice([0.0, 0.1], 1500), rng.random(1500))
