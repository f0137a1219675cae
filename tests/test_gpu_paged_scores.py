"""Attention over pages whose scores are so large that an f32 holds no fraction of them: what is equal weighs the same, the largest takes
all, and nothing overflows on the way, in both attentions."""
import numpy as np
import pytest

import paged_ref as ref
from test_gpu_paged import OnDevice

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("power", [10, 20, 24, 25, 26, 27, 30, 35, 60, 100])
def test_attention_with_scores_beyond_the_fractions_of_f32(ex, hd, sign, power):
    """Queries and keys of one element that is not zero, in whole powers of two times 3 or 5: every score is exact but for the one
    constant that all share, so equal scores are equal in any arithmetic and others lie hundreds apart.  A row is then the mean of
    the values at its largest score: n products and sums, a quotient and the weights' own rounding, (n + 40) steps of f32 twice."""
    print("scores", hd, sign, power, flush=True)
    rng = np.random.default_rng(hd + power)
    prior, new, n_kv, group = 90, 70, 1, 3
    b = ref.Batch(rng, [prior + new, 45], 16, n_kv, hd, [new, 45])
    b.k[:] = 0
    levels = np.array([3.0, 2.5, 2.0, 1.0])
    where = {}
    for s in range(2):
        lv = rng.choice(4, int(b.kv_len[s]), p=[0.05, 0.25, 0.3, 0.4])
        lv[0] = 1                                                # the largest so far changes on the way
        where[s] = lv
        for p in range(int(b.kv_len[s])):
            b.k[b.table[s, p // 16], 0, p % 16, 5] = sign * levels[lv[p]]
    n_heads = n_kv * group
    q = np.zeros((new + 45, n_heads, hd), dtype=np.float32)
    q[:, :, 5] = 2.0 ** power * np.array([1.0, 3.0, 5.0])
    d = OnDevice(ex, b)
    dq, dout = ex.to_device(q.reshape(len(q), -1)), ex.buffer(q.nbytes)
    ex.paged_attn_prefill_dev(d.pool, d.seqs, dq, len(q), n_heads, dout)
    pre = dout.download(np.float32).reshape(q.shape)
    last = np.stack([q[new - 1], q[-1]])
    ex.paged_attn_decode_dev(d.pool, d.seqs, ex.to_device(last), n_heads, dout)
    dec = dout.download(np.float32, last.size).reshape(last.shape)

    def check(got, s, n, what):
        _, _, v = b.rows(s, 0, n)
        at = sign * levels[where[s][:n]]
        if power < 20:                                           # a gap of half a level is then no more than hundreds
            assert 0.5 * 2.0 ** power / hd ** 0.5 > 40
        on = at == at.max()
        want, bound = v[on].mean(0), 2 * (n + 40) * ref.U32 * np.abs(v[on]).mean(0) + 1e-30
        assert (np.abs(got - want) <= bound).all(), (what, s, n, float((np.abs(got - want) / bound).max()), int(on.sum()))

    for t, s, pos in b.places():
        check(pre[t], s, pos + 1, "prefill")
    for s in range(2):
        check(dec[s], s, int(b.kv_len[s]), "decode")
