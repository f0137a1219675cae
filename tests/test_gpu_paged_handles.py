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


def test_distances_between_rows_that_lead_out_of_a_buffer_are_refused(ex):
    """A negative distance (which a size_t takes for a huge one), and one of more floats than any buffer has."""
    from rustorch_amd.errors import ShapeMismatch
    kv = ex.paged_kv(8, 16, 1, 64)
    table, ones = ex.to_device(np.arange(8, dtype=np.int32)), ex.to_device(np.full(4, 3, dtype=np.int32))
    cu = ex.to_device(np.arange(5, dtype=np.int32))
    seqs = ex.paged_seqs(table, ones, 4, 2, cu, 3)
    x = ex.to_device(np.ones(4096, dtype=np.float32))
    u, token = ex.to_device(np.full(4, 0.5)), ex.to_device(np.zeros(4, dtype=np.int32))
    for ld in (-4, -64, -2 ** 40, 60, 2 ** 62, 2 ** 63 - 4):
        for kw in (dict(k_ld=ld), dict(v_ld=ld), dict(q_ld=ld), dict(q_out_ld=ld)):
            with pytest.raises(ShapeMismatch):
                ex.paged_append_dev(kv, seqs, x, x, 4, q=x, q_out=x, n_heads=1, **kw)
        for call in (ex.paged_attn_decode_dev, lambda kv, seqs, q, h, out, **kw: ex.paged_attn_prefill_dev(kv, seqs, q, 4, h, out, **kw)):
            for kw in (dict(q_ld=ld), dict(out_ld=ld)):
                with pytest.raises(ShapeMismatch):
                    call(kv, seqs, x, 1, x, **kw)
        with pytest.raises(ShapeMismatch):
            ex.sample_dev(x, 4, 64, u, token, ld=ld)
    lib, wrapped = ex.lib, 2 ** 64 - 4
    assert lib.rt_hip_paged_append_dev(ex.ctx, kv.handle, table.ptr, 2, ones.ptr, cu.ptr, 4, 4, x.ptr, wrapped, x.ptr, 64, None, 0, None, 0, 0, 0, 1.0) == 2
    assert lib.rt_hip_paged_attn_decode_dev(ex.ctx, kv.handle, table.ptr, 2, ones.ptr, 4, 3, x.ptr, wrapped, 1, x.ptr, 64) == 2
    assert lib.rt_hip_paged_attn_prefill_dev(ex.ctx, kv.handle, table.ptr, 2, ones.ptr, cu.ptr, 4, 4, x.ptr, 64, 1, x.ptr, wrapped) == 2
    assert lib.rt_hip_sample_dev(ex.ctx, x.ptr, wrapped, 4, 64, None, None, None, None, u.ptr, token.ptr, None) == 2
    ex.synchronize()
