"""An executor on a stream of the caller's: its calls run in the order of torch's work on that stream, with no host wait between, and a
capture of that stream either holds them or refuses them."""
import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs torch on the device", allow_module_level=True)

from rustorch_amd.errors import InvalidParameters  # noqa: E402
from rustorch_amd.executor import HipKernelExecutor  # noqa: E402

BUSY = 20_000_000          # device clocks that a stream is kept busy for before the inputs are written: some milliseconds


def borrowed(ex, t):
    return ex.borrow(t.data_ptr(), t.numel() * t.element_size())


@pytest.mark.parametrize("which", ["default", "side"])
def test_calls_run_in_the_order_of_the_callers_stream(which):
    """Logits that a busy stream writes late are the ones that are sampled, and what torch reads behind the call is its answer; the
    inputs change again right behind it."""
    print("order of the stream", which, flush=True)
    stream = torch.cuda.default_stream() if which == "default" else torch.cuda.Stream()
    rows, vocab = 4, 50000
    g = torch.Generator().manual_seed(1)
    with torch.cuda.stream(stream), HipKernelExecutor(0, stream=stream.cuda_stream) as ex:
        want = [torch.randint(0, vocab, (rows,), generator=g) for _ in range(5)]
        late = [torch.nn.functional.one_hot(w, vocab).float().cuda() for w in want]
        x, u = torch.zeros(rows, vocab, device="cuda"), torch.full((rows,), 0.5, dtype=torch.float64, device="cuda")
        token, temp = torch.full((rows,), -7, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
        bx, bu, bt, btemp = (borrowed(ex, t) for t in (x, u, token, temp))
        ex.sample_dev(bx, rows, vocab, bu, bt, temperature=btemp)          # the workspace is there
        got = []
        torch.cuda.synchronize()
        for t in late:
            torch.cuda._sleep(BUSY)
            x.copy_(t)
            ex.sample_dev(bx, rows, vocab, bu, bt, temperature=btemp)
            got.append(token.clone())
            x.zero_()
            token.fill_(-7)
        stream.synchronize()
        assert [t.tolist() for t in got] == [w.tolist() for w in want]


def test_several_executors_on_one_stream_and_their_ends():
    """Executors come and go on a stream that stays the caller's."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        a = torch.arange(8, dtype=torch.float32, device="cuda")
        for i in range(3):
            with HipKernelExecutor(0, stream=stream.cuda_stream) as ex, HipKernelExecutor(0, stream=stream.cuda_stream) as other:
                for e in (ex, other):
                    e.add_dev(borrowed(e, a), borrowed(e, a), 8)
            assert a.tolist() == [v * 4.0 ** (i + 1) for v in range(8)]


def paged_case(rng, n_seq_len, new, n_kv, n_heads, hd):
    b = ref.Batch(rng, n_seq_len, 16, n_kv, hd, new)
    t = dict(table=b.table, kv_len=b.kv_len, cu=b.cu, k=b.k, v=b.v, q=rng.standard_normal((sum(new), n_heads * hd)).astype(np.float32))
    return b, {k: torch.from_numpy(np.ascontiguousarray(x)).cuda() for k, x in t.items()}


def test_a_capture_of_the_callers_stream_holds_calls_without_a_workspace():
    """Append and prefill attention captured once, replayed on inputs that change between the replays, with work outside the graph
    between them: every replay equals the eager calls."""
    rng = np.random.default_rng(7)
    n_kv, n_heads, hd = 2, 4, 64
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), HipKernelExecutor(0, stream=stream.cuda_stream) as ex:
        b, t = paged_case(rng, [40, 5], [9, 5], n_kv, n_heads, hd)
        k, v = (torch.randn(14, n_kv * hd, device="cuda") for _ in range(2))
        qr, out = torch.zeros_like(t["q"]), torch.zeros_like(t["q"])
        pool = ex.wrap_paged_kv(borrowed(ex, t["k"]), borrowed(ex, t["v"]), b.n_pages, 16, n_kv, hd)
        seqs = ex.paged_seqs(borrowed(ex, t["table"]), borrowed(ex, t["kv_len"]), 2, b.max_blocks, borrowed(ex, t["cu"]))
        bk, bv, bq, bqr, bout = (borrowed(ex, x) for x in (k, v, t["q"], qr, out))

        def step():
            ex.paged_append_dev(pool, seqs, bk, bv, 14, q=bq, q_out=bqr, n_heads=n_heads)
            ex.paged_attn_prefill_dev(pool, seqs, bqr, 14, n_heads, bout)

        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for i in range(4):
            for x in (k, v, t["q"]):
                x.normal_()
            out.zero_()
            graph.replay()
            replayed, pages = out.clone(), t["k"].clone()
            out.zero_()
            t["k"].view(torch.int16)[:, :, 5:7] ^= 0                       # work of the caller's own
            step()
            stream.synchronize()
            assert torch.equal(replayed, out) and torch.equal(pages, t["k"]) and bool((out != 0).any())


def test_a_capture_of_the_callers_stream_refuses_what_it_cannot_keep():
    """A split decode step and a large sampling need the workspace, which may move later; a memset is no part of a graph here.  The
    capture goes on without them, and the calls work before and behind it."""
    rng = np.random.default_rng(8)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), HipKernelExecutor(0, stream=stream.cuda_stream) as ex:
        b, t = paged_case(rng, [1500, 30], [1, 1], 1, 2, 64)
        pool = ex.wrap_paged_kv(borrowed(ex, t["k"]), borrowed(ex, t["v"]), b.n_pages, 16, 1, 64)
        seqs = ex.paged_seqs(borrowed(ex, t["table"]), borrowed(ex, t["kv_len"]), 2, b.max_blocks, None, 1500)
        out = torch.zeros_like(t["q"])
        x, u, token = torch.zeros(2, 40000, device="cuda"), torch.zeros(2, dtype=torch.float64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
        bq, bout, bx, bu, bt = (borrowed(ex, y) for y in (t["q"], out, x, u, token))
        a = torch.ones(4, device="cuda")
        ba = borrowed(ex, a)
        ex.paged_attn_decode_dev(pool, seqs, bq, 2, bout)
        first = out.clone()
        stream.synchronize()
        graph, refused = torch.cuda.CUDAGraph(), 0
        with torch.cuda.graph(graph, stream=stream):
            for call in (lambda: ex.paged_attn_decode_dev(pool, seqs, bq, 2, bout), lambda: ex.sample_dev(bx, 2, 40000, bu, bt), lambda: bout.zero()):
                try:
                    call()
                except InvalidParameters as e:
                    refused += "capture" in str(e)
            ex.add_dev(ba, ba, 4)
        assert refused == 3
        for i in range(3):
            graph.replay()
            out.zero_()
            ex.paged_attn_decode_dev(pool, seqs, bq, 2, bout)
            stream.synchronize()
            assert torch.equal(out, first) and a.tolist() == [2.0 ** (i + 1)] * 4


CFG = dict(n_layers=2, hidden=256, n_heads=2, ffn=512, vocab=128, max_pos=24)


def walk(ex, mode):
    """Picks and logits of a small model over a prompt, steps and a decode."""
    from rustorch_amd import llama
    m = llama.HipLlama(ex, **CFG)
    llama.load_synthetic(m, 5)
    m.set_mode(mode)
    m.prefill([3, 77, 100, 9, 14], 0)
    picks = [m.step(t, 5 + i) for i, t in enumerate((1, 2, 3, 4))]
    out = picks, m.decode(picks[-1], 9, 6).tolist(), m.logits()
    m.close()
    return out


@pytest.mark.parametrize("which,mode", [("default", 1), ("side", 1), ("side", 2)])
def test_a_model_on_the_callers_stream(ex, which, mode):
    """The same picks and logits, bit for bit, as on a stream of the executor's own."""
    stream = torch.cuda.default_stream() if which == "default" else torch.cuda.Stream()
    want = walk(ex, 1)
    with torch.cuda.stream(stream), HipKernelExecutor(0, stream=stream.cuda_stream) as mine:
        got = walk(mine, mode)
    assert got[:2] == want[:2] and np.array_equal(got[2], want[2])


def test_a_model_refuses_the_graphs_that_cannot_be():
    """Mode 2 on the default stream, which cannot be captured, and a step inside a capture of the caller's, whose replays would not count
    the tokens; the model goes on as before."""
    from rustorch_amd import llama
    with HipKernelExecutor(0, stream=0) as mine:
        m = llama.HipLlama(mine, **CFG)
        with pytest.raises(InvalidParameters, match="default stream"):
            m.set_mode(2)
        m.close()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), HipKernelExecutor(0, stream=stream.cuda_stream) as mine:
        m = llama.HipLlama(mine, **CFG)
        llama.load_synthetic(m, 5)
        b = llama.HipLlamaBatch(m, 3, 24)
        first = m.step(3, 0)
        a = torch.ones(4, device="cuda")
        ba = borrowed(mine, a)
        graph, refused = torch.cuda.CUDAGraph(), 0
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            for call in (lambda: m.step(7, 1, want_token=False), lambda: m.prefill([1, 2, 3], 1), lambda: m.decode(1, 1, 2), lambda: b.step([1, 2, 3], [0, 0, 0], want_tokens=False),
                         lambda: b.prefill(0, [1, 2, 3])):
                try:
                    call()
                except InvalidParameters as e:
                    refused += "capture" in str(e)
            mine.add_dev(ba, ba, 4)
        graph.replay()
        stream.synchronize()
        assert refused == 5 and a.tolist() == [2.0] * 4
        m.step(7, 1)
        got = m.logits()
        m.reset()
        assert m.step(3, 0) == first
        m.step(7, 1)
        assert np.array_equal(m.logits(), got)
        b.close()
        m.close()


def test_a_captured_step_of_short_sequences(ex):
    """A whole decode step without a workspace (append, attention of up to 256 positions, sampling of a small vocabulary) replayed with
    lengths and tokens that the device moves on: each replay equals the eager calls of another executor."""
    rng = np.random.default_rng(9)
    n_seq, n_kv, n_heads, hd, vocab = 3, 2, 4, 64, 4 * 64
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), HipKernelExecutor(0, stream=stream.cuda_stream) as mine:
        b, t = paged_case(rng, [200, 17, 90], [1, 1, 1], n_kv, n_heads, hd)
        other = {k: x.clone() for k, x in t.items()}
        kv = [torch.randn(n_seq, n_kv * hd, device="cuda") for _ in range(2)]
        u = torch.rand(n_seq, dtype=torch.float64, device="cuda")
        start = t["kv_len"].clone() - 8
        outs = []

        def calls(e, t):
            pool = e.wrap_paged_kv(borrowed(e, t["k"]), borrowed(e, t["v"]), b.n_pages, 16, n_kv, hd)
            seqs = e.paged_seqs(borrowed(e, t["table"]), borrowed(e, t["kv_len"]), n_seq, b.max_blocks, None, 208)
            out, token = torch.zeros_like(t["q"]), torch.zeros(n_seq, dtype=torch.int32, device="cuda")
            bk, bv, bu, bq, bout, btok = (borrowed(e, x) for x in (*kv, u, t["q"], out, token))

            def step():
                e.paged_append_dev(pool, seqs, bk, bv, n_seq, q=bq, q_out=bout, n_heads=n_heads)
                e.paged_attn_decode_dev(pool, seqs, bout, n_heads, bout)
                e.sample_dev(bout, n_seq, vocab, bu, btok)

            return step, out, token

        graph_step, out, token = calls(mine, t)
        eager_step, out2, token2 = calls(ex, other)
        graph = torch.cuda.CUDAGraph()
        graph_step()                                                       # both once before the capture: it stores keys, too
        stream.synchronize()
        eager_step()
        ex.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            graph_step()
        for x in (t, other):
            x["kv_len"].copy_(start)
        for i in range(5):
            for x in (*kv, t["q"]):
                x.normal_()
            other["q"].copy_(t["q"])
            u.uniform_()
            for x in (t, other):
                x["kv_len"] += 1
            graph.replay()
            stream.synchronize()                                           # ex has a stream of its own: the host waits for both
            eager_step()
            ex.synchronize()
            outs.append((out.clone(), token.clone()))
            assert torch.equal(out, out2) and torch.equal(token, token2) and torch.equal(t["k"], other["k"])
        assert not torch.equal(outs[0][0], outs[1][0])


def test_two_threads_on_one_executor(ex):
    """Split decode steps of two batches from two host threads: the calls take turns on the context and its workspace."""
    import threading
    rng = np.random.default_rng(10)
    work, errors = [], []
    for lens in ([2500, 3], [40, 900, 1700]):
        b = ref.Batch(rng, lens, 16, 2, 64)
        pool = ex.paged_kv(b.n_pages, 16, 2, 64)
        k, v = pool.pages()
        k.upload(b.k.view(np.uint16)), v.upload(b.v.view(np.uint16))
        seqs = ex.paged_seqs(ex.to_device(b.table), ex.to_device(b.kv_len), b.n_seq, b.max_blocks, None, max(lens))
        q = rng.standard_normal((b.n_seq, 4 * 64)).astype(np.float32)
        work.append((pool, seqs, ex.to_device(q), [ex.buffer(q.nbytes) for _ in range(40)], ex.buffer(q.nbytes)))
    for pool, seqs, q, outs, first in work:
        ex.paged_attn_decode_dev(pool, seqs, q, 4, first)

    def loop(pool, seqs, q, outs, first):
        try:
            for o in outs:
                ex.paged_attn_decode_dev(pool, seqs, q, 4, o)
        except Exception as e:      # noqa: BLE001  (reported by the main thread)
            errors.append(e)

    threads = [threading.Thread(target=loop, args=w) for w in work]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors
    for _, _, _, outs, first in work:
        want = first.download(np.float32)
        assert np.isfinite(want).all() and all(np.array_equal(o.download(np.float32), want) for o in outs)
