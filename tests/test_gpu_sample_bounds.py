"""Sampling at the least probability that the header says can be drawn, on both launch forms."""
import math

import numpy as np
import pytest

from test_gpu_sample import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [3, 2048, 2049, 32000, 40000, 131072, 131073, 1 << 20])
def test_the_least_probability_that_can_be_drawn(ex, vocab):
    """Token 0 a little more and a little less likely than 2^-(F + 1) of the last one, u = 0: the first token that can be drawn at all.
    A step of half a power of two is 0.35 in the logits, 1e5 times what f32 rounds them by."""
    print("least probability", vocab, flush=True)
    f = min(51, 62 - math.ceil(math.log2(vocab)))
    x = np.full((2, vocab), -np.inf)
    x[:, -1] = 0.0
    x[0, 0], x[1, 0] = -(f + 0.5) * math.log(2), -(f + 1.5) * math.log(2)
    for kw in (dict(), dict(top_k=2)):
        tok, prob = run(ex, x, u=0.0, **kw)
        assert tok.tolist() == [0, vocab - 1], (kw, tok)
        assert prob[1] == 1.0 and abs(prob[0] / 2.0 ** -(f + 0.5) - 1) < 1e-4
