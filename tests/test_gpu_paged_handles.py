"""What the paged operators' Python handles keep alive and refuse (host logic; the calls that are refused launch nothing)."""
import gc
import weakref

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_page_buffers_keep_their_pool(ex):
    """The buffers of pages() are of use after the pool's own name is gone: the pool is freed with the last of them."""
    k, v = ex.paged_kv(3, 16, 2, 64).pages()
    gc.collect()
    x = np.arange(k.nbytes // 2, dtype=np.uint16)
    k.upload(x)
    v.upload(x[::-1].copy())
    assert np.array_equal(k.download(np.uint16), x) and np.array_equal(v.download(np.uint16), x[::-1])
    pool = ex.paged_kv(2, 16, 1, 64)
    gone = weakref.ref(pool)
    k, v = pool.pages()
    wrapped = ex.wrap_paged_kv(k, v, 2, 16, 1, 64)               # a pool over those pages keeps them too
    del pool, k, v
    gc.collect()
    assert gone() is not None
    wrapped.pages()[0].upload(np.zeros(2 * 16 * 64, dtype=np.uint16))
    del wrapped
    gc.collect()
    assert gone() is None


def test_a_borrowed_view_keeps_what_it_is_told_to(ex):
    whole = ex.to_device(np.arange(64, dtype=np.float32))
    gone = weakref.ref(whole)
    view = ex.borrow(whole.ptr.value + 4 * 32, 4 * 32, keep=whole)
    del whole
    gc.collect()
    assert gone() is not None and np.array_equal(view.download(np.float32), np.arange(32, 64, dtype=np.float32))
    view.free()
    gc.collect()
    assert gone() is None
