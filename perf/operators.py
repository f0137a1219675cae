"""What the serving operators are measured on: the cases, their plain forms, and the calls a user makes.

Four operators of a server that keeps the keys and values of many sequences in pages of one pool:

- ``append``: the new tokens' queries and keys are rotated by their positions, keys and values go to the pages (fp16);
- ``decode``: one new query per sequence attends its sequence's pages;
- ``prefill``: several new queries per sequence attend its pages, each up to its own position;
- ``sample``: one token per row of logits, by temperature, top-k, top-p and min-p, from given random numbers.

Pages are ``[n_pages][n_kv_heads][page_size][head_dim]`` halves, one pool for the keys and one for the values; position p of
sequence s is slot ``p % page_size`` of page ``table[s][p // page_size]``.  Activations are f32.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
_ex = {}


def _executor():
    """One executor for the process, as a server has, on the stream that makes the inputs and reads the outputs: its calls run in
    the order of torch's work."""
    stream = torch.cuda.current_stream().cuda_stream
    if stream not in _ex:
        from rustorch_amd.executor import HipKernelExecutor
        _ex[stream] = HipKernelExecutor(0, stream=stream)
    return _ex[stream]


# ------------------------------------------------------------------------------------------------------------ the cases


def listed():
    head = dict(heads=32, kv=32, hd=128)          # the 7B shape of the benchmark
    gqa = dict(heads=32, kv=8, hd=128)
    return [
        # the append of one decode step of one sequence: latency
        dict(name="append one", op="append", n_seq=1, new_lo=1, new_hi=1, prior_lo=1999, prior_hi=1999, page=16, rope="interleaved", theta=10000.0, **head),
        # prompts of very different lengths arriving together, some behind a cached prefix
        dict(name="append ragged", op="append", n_seq=7, new_lo=1, new_hi=4095, prior_lo=0, prior_hi=1001, page=64, rope="half", theta=500000.0, **gqa),
        # the benchmark's single chat: few positions, every head with keys of its own
        dict(name="decode one short", op="decode", n_seq=1, len_lo=200, len_hi=200, page=16, **head),
        # a small model's heads, sequences that have not begun among them
        dict(name="decode small heads", op="decode", n_seq=9, len_lo=0, len_hi=1501, page=128, heads=12, kv=12, hd=64),
        # an ordinary continuous batch
        dict(name="decode ragged batch", op="decode", n_seq=33, len_lo=1, len_hi=4097, page=16, **gqa),
        # one document: the length is all the parallelism there is
        dict(name="decode one long", op="decode", n_seq=1, len_lo=131071, len_hi=131071, page=64, **gqa),
        # a full server
        dict(name="decode full server", op="decode", n_seq=48, len_lo=1000, len_hi=16000, page=32, heads=32, kv=4, hd=128),
        # the benchmark's prompt
        dict(name="prefill one", op="prefill", n_seq=1, new_lo=512, new_hi=512, prior_lo=0, prior_hi=0, page=16, **head),
        # chunks of prompts behind prefixes of every length, down to one token
        dict(name="prefill ragged", op="prefill", n_seq=6, new_lo=1, new_hi=701, prior_lo=0, prior_hi=3001, page=16, **gqa),
        # a long document in one pass
        dict(name="prefill long", op="prefill", n_seq=1, new_lo=8191, new_hi=8191, prior_lo=0, prior_hi=0, page=64, **gqa),
        # one chat's next token over the benchmark's vocabulary
        dict(name="sample one", op="sample", rows=1, vocab=32000, temperature=0.8, top_k=40, top_p=0.95, min_p=0.0, mixed=False),
        # a batch in which every request brings its own settings, over a large odd vocabulary
        dict(name="sample mixed batch", op="sample", rows=77, vocab=131071, temperature=1.0, top_k=0, top_p=0.9, min_p=0.0, mixed=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prefill", "sample"])
    if op == "sample":
        vocab = _log(rng, 1000, 150000)
        rows = _log(rng, 1, min(128, 10000000 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]), top_k=rng.choice([0, 0, 1, 2, 17, 50, 333, 1500]),
                    top_p=rng.choice([0.0, 0.1, 0.5, 0.9, 0.95, 0.999, 1.0]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1, 0.5]), mixed=rng.random() < 0.3)
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    group = rng.choice([1, 2, 3, 4, 5, 8, 12])
    while kv * group > 48:
        group = max(1, group // 2)
    c = dict(op=op, heads=kv * group, kv=kv, hd=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128, 256]))
    if op == "decode":
        longest = _log(rng, 1, 100000)
        c["n_seq"] = _log(rng, 1, max(1, min(128, 1500000 // (longest * kv))))
        c["len_hi"], c["len_lo"] = longest, rng.choice([0, 1, longest // 3, longest])
    else:
        most = 3500 if op == "prefill" else 8000
        new = _log(rng, 1, most)
        c["n_seq"] = _log(rng, 1, max(1, min(64, most // new)))
        c["new_hi"], c["new_lo"] = new, rng.choice([0, 1, new // 2, new])
        c["prior_hi"] = rng.choice([0, _log(rng, 1, 4000)])
        c["prior_lo"] = rng.choice([0, c["prior_hi"] // 2])
        if op == "append":
            c["rope"], c["theta"] = rng.choice(["interleaved", "half"]), rng.choice([10000.0, 500000.0])
    return c


def _spread(lo, hi, n):
    """n whole numbers from lo to hi in even steps (the largest alone for n = 1)."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lengths(c):
    """(new tokens, positions with the new ones) of each sequence: the same for every seed."""
    n = c["n_seq"]
    if c["op"] == "decode":
        kv = _spread(c["len_lo"], c["len_hi"], n)
        return [min(1, x) for x in kv], kv
    new = _spread(c["new_lo"], c["new_hi"], n)
    prior = _spread(c["prior_lo"], c["prior_hi"], n)[::-1]
    return new, [a + b for a, b in zip(new, prior)]


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 32 * case["rows"], "flops": 4 * n}
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    new, length = _lengths(case)
    if case["op"] == "append":          # q in and out, k and v in as f32 and out as halves
        t = sum(new)
        return {"bytes": t * hd * (8 * h + 12 * kv), "flops": t * hd * 3 * (h + kv)}
    q = case["n_seq"] if case["op"] == "decode" else sum(new)
    seen = sum(length) if case["op"] == "decode" else sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, length))
    return {"bytes": 4 * kv * hd * sum(length) + 8 * q * h * hd, "flops": 4 * h * hd * seen}


# ----------------------------------------------------------------------------------------------------------- the inputs


def _sample_inputs(c, g):
    n, v = c["rows"], c["vocab"]
    logits = torch.randn(n, v, generator=g, device=DEV) * 2.0
    peak = torch.randint(0, v, (n, 64), generator=g, device=DEV)          # the tokens that the context asks for
    logits.scatter_add_(1, peak, torch.rand(n, 64, generator=g, device=DEV) * 8.0)
    row = torch.arange(n)
    pick = lambda values, step: torch.tensor(values)[(row // step) % len(values)] if c["mixed"] else torch.tensor(values[:1]).expand(n)  # noqa: E731
    st = dict(logits=logits,
              temperature=pick([c["temperature"], 0.7, 0.0, 1.3], 1).to(torch.float32).to(DEV).contiguous(),
              top_k=pick([c["top_k"], 40, 400], 1).to(torch.int32).to(DEV).contiguous(),
              top_p=pick([c["top_p"], 0.95, 1.0], 3).to(torch.float32).to(DEV).contiguous(),
              min_p=pick([c["min_p"], 0.05], 5).to(torch.float32).to(DEV).contiguous(),
              u=torch.rand(n, generator=g, device=DEV, dtype=torch.float64),
              token=torch.zeros(n, dtype=torch.int32, device=DEV), prob=torch.zeros(n, device=DEV))
    return st


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    c = dict(case)
    if c["op"] == "sample":
        st = _sample_inputs(c, g)
    else:
        new, length = _lengths(c)
        n, h, kv, hd, ps = c["n_seq"], c["heads"], c["kv"], c["hd"], c["page"]
        blocks = [-(-x // ps) for x in length]
        wide = max(1, max(blocks))
        n_pages = sum(blocks) + 3
        order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
        first = torch.tensor([sum(blocks[:i]) for i in range(n)], device=DEV)
        many = torch.tensor(blocks, device=DEV)
        j = torch.arange(wide, device=DEV)
        table = torch.where(j < many[:, None], order[(first[:, None] + j).clamp(max=n_pages - 1)], -1).to(torch.int32).contiguous()
        rows = n if c["op"] == "decode" else sum(new)
        cu = torch.tensor([sum(new[:i]) for i in range(n + 1)], dtype=torch.int32, device=DEV)
        pool = lambda: torch.randn(n_pages, kv, ps, hd, generator=g, device=DEV, dtype=torch.float16)  # noqa: E731
        st = dict(table=table, kv_len=torch.tensor(length, dtype=torch.int32, device=DEV), cu=cu, k_pages=pool(), v_pages=pool(),
                  q=torch.randn(rows, h * hd, generator=g, device=DEV) * 2.0, out=torch.zeros(rows, h * hd, device=DEV), longest=max(length), most_new=max(new))
        if c["op"] == "append":
            st["k"], st["v"] = (torch.randn(rows, kv * hd, generator=g, device=DEV) for _ in range(2))
    st["case"] = c
    if own:
        _wrap(st)
    return st


def _wrap(st):
    """The handles that a user's program keeps: device buffers over the tensors, the page pool, the batch's description."""
    st["ex"], c = _executor(), st["case"]
    ex = st["ex"]
    st["buf"] = b = {k: ex.borrow(t.data_ptr(), t.numel() * t.element_size()) for k, t in st.items() if isinstance(t, torch.Tensor)}
    if c["op"] != "sample":
        st["pool"] = ex.wrap_paged_kv(b["k_pages"], b["v_pages"], st["k_pages"].shape[0], c["page"], c["kv"], c["hd"])
        st["seqs"] = ex.paged_seqs(b["table"], b["kv_len"], c["n_seq"], st["table"].shape[1], None if c["op"] == "decode" else b["cu"], st["longest"])


# ------------------------------------------------------------------------------------------------------- the plain forms


def _token_places(st):
    """(sequence, position) of each new token's row."""
    t = torch.arange(st["q"].shape[0], device=DEV)
    seq = torch.searchsorted(st["cu"][1:].long(), t, right=True)
    return seq, st["kv_len"].long()[seq] - st["cu"].long()[seq + 1] + t


def _angles(pos, hd, theta):
    freq = theta ** (-2.0 * torch.arange(hd // 2, device=DEV, dtype=torch.float64) / hd)
    a = pos.double()[:, None] * freq
    return a.cos(), a.sin()


def _turn(x, cos, sin, style):
    """x [rows, heads, hd] turned pair by pair; cos, sin [rows, hd / 2]."""
    cos, sin = cos[:, None, :], sin[:, None, :]
    if style == "half":
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _plain_append(st):
    c = st["case"]
    seq, pos = _token_places(st)
    cos, sin = _angles(pos, c["hd"], c["theta"])
    cos, sin = cos.float(), sin.float()
    heads = lambda x: x.view(x.shape[0], -1, c["hd"])  # noqa: E731
    st["out"].copy_(_turn(heads(st["q"]), cos, sin, c["rope"]).flatten(1))
    page, slot = st["table"][seq, pos // c["page"]].long(), pos % c["page"]
    st["k_pages"][page, :, slot] = _turn(heads(st["k"]), cos, sin, c["rope"]).half()
    st["v_pages"][page, :, slot] = heads(st["v"]).half()
    return {"q": st["out"], "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


def _rows_of(pages, table):
    """The pages of every sequence one behind the other, in f32: [sequences, kv heads, positions, hd]."""
    x = pages[table.long().clamp(min=0)]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3).float()


def _attend(q, k, v, seen):
    """q [s, kv, rows, hd] over k, v [s, kv, positions, hd]; seen [s, 1, rows or 1, positions] says which."""
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(q.shape[-1]))
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isinf(top), 0.0, top))
    total = e.sum(-1, keepdim=True)
    return torch.matmul(e, v) / torch.where(total == 0, 1.0, total)


def _plain_decode(st):
    c = st["case"]
    n, kv, hd = c["n_seq"], c["kv"], c["hd"]
    k, v = _rows_of(st["k_pages"], st["table"]), _rows_of(st["v_pages"], st["table"])
    seen = (torch.arange(k.shape[2], device=DEV) < st["kv_len"][:, None])[:, None, None, :]
    v = torch.where(seen.transpose(-1, -2), v, 0.0)
    st["out"].copy_(_attend(st["q"].view(n, kv, -1, hd), k, v, seen).reshape(n, -1))
    return st["out"]


def _plain_prefill(st):
    c = st["case"]
    n, kv, hd, wide = c["n_seq"], c["kv"], c["hd"], st["most_new"]
    group = c["heads"] // kv
    k, v = _rows_of(st["k_pages"], st["table"]), _rows_of(st["v_pages"], st["table"])
    j = torch.arange(k.shape[2], device=DEV)
    v = torch.where((j < st["kv_len"][:, None])[:, None, :, None], v, 0.0)
    seq, pos = _token_places(st)
    nth = torch.arange(seq.shape[0], device=DEV) - st["cu"].long()[seq]
    q = torch.zeros(n, wide, c["heads"] * hd, device=DEV)
    q[seq, nth] = st["q"]
    at = torch.full((n, wide), -1, device=DEV)
    at[seq, nth] = pos
    q = q.view(n, wide, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, group * wide, hd)
    seen = (j <= at[:, :, None])[:, None, None].expand(n, 1, group, wide, j.numel()).reshape(n, 1, group * wide, j.numel())
    o = _attend(q, k, v, seen).view(n, kv, group, wide, hd).permute(0, 3, 1, 2, 4).reshape(n, wide, -1)
    st["out"].copy_(o[seq, nth])
    return st["out"]


def _plain_sample(st):
    x = st["logits"]
    n, vocab = x.shape
    t, k, p, low = (st[name][:, None] for name in ("temperature", "top_k", "top_p", "min_p"))
    greedy = (t <= 0) | (k == 1)
    ordered, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((ordered.double() - ordered[:, :1].double()) / torch.where(greedy, 1.0, t).double())
    nth = torch.arange(vocab, device=DEV)
    w = torch.where((nth < torch.where(k <= 0, vocab, k)) & (~greedy | (nth == 0)), w, 0.0)
    before = torch.cumsum(w, -1) - w
    p = torch.where((p <= 0) | (p >= 1), 2.0, p).double()
    w = torch.where((before < p * w.sum(-1, keepdim=True)) & (w >= low.double()), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    run_up = torch.cumsum(w, -1)
    total = run_up[:, -1:]
    tok = torch.argmax(((run_up > st["u"][:, None] * total) & (w > 0)).to(torch.uint8), -1, keepdim=True)
    st["token"].copy_(tok[:, 0])
    st["prob"].copy_((w.gather(1, tok) / total)[:, 0])
    return {"token": st["token"], "prob": st["prob"]}


_PLAIN = {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill, "sample": _plain_sample}


# ---------------------------------------------------------------------------------------------------- the user's calls


def run(state):
    c = state["case"]
    if not own:
        return _PLAIN[c["op"]](state)
    ex, b = state["ex"], state["buf"]
    if c["op"] == "append":
        ex.paged_append_dev(state["pool"], state["seqs"], b["k"], b["v"], state["q"].shape[0], q=b["q"], q_out=b["out"], n_heads=c["heads"], rope=c["rope"], theta=c["theta"])
        return {"q": state["out"], "k_pages": state["k_pages"], "v_pages": state["v_pages"]}
    if c["op"] == "decode":
        ex.paged_attn_decode_dev(state["pool"], state["seqs"], b["q"], c["heads"], b["out"])
        return state["out"]
    if c["op"] == "prefill":
        ex.paged_attn_prefill_dev(state["pool"], state["seqs"], b["q"], state["q"].shape[0], c["heads"], b["out"])
        return state["out"]
    ex.sample_dev(b["logits"], c["rows"], c["vocab"], b["u"], b["token"], temperature=b["temperature"], top_k=b["top_k"], top_p=b["top_p"], min_p=b["min_p"], out_prob=b["prob"])
    return {"token": state["token"], "prob": state["prob"]}


# ------------------------------------------------------------------------------------ the definitions, in 64 bits


def _exact_append(st):
    c = st["case"]
    hd, half = c["hd"], c["hd"] // 2
    new, length = _lengths(c)
    out, kp, vp = st["q"].double(), st["k_pages"].double(), st["v_pages"].double()
    first = torch.arange(half, device=DEV) * (1 if c["rope"] == "half" else 2)
    second = first + (half if c["rope"] == "half" else 1)
    at = 0
    for s, (n, total) in enumerate(zip(new, length)):
        if n == 0:
            continue
        pos = torch.arange(total - n, total, device=DEV)
        turn = torch.polar(torch.ones(n, half, device=DEV, dtype=torch.float64),
                           torch.outer(pos.double(), torch.exp(-math.log(c["theta"]) * 2.0 / hd * torch.arange(half, device=DEV, dtype=torch.float64))))
        for name, heads in (("q", c["heads"]), ("k", c["kv"])):
            x = st[name][at:at + n].double().view(n, heads, hd)
            z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
            y = torch.empty_like(x)
            y[..., first], y[..., second] = z.real, z.imag
            if name == "q":
                out[at:at + n] = y.reshape(n, -1)
            else:
                kp[st["table"][s].long()[pos // c["page"]], :, pos % c["page"]] = y
        vp[st["table"][s].long()[pos // c["page"]], :, pos % c["page"]] = st["v"][at:at + n].double().view(n, c["kv"], hd)
        at += n
    return {"q": out, "k_pages": kp, "v_pages": vp}


def _exact_attention(st):
    c = st["case"]
    new, length = _lengths(c)
    if c["op"] == "decode":
        new = [1] * c["n_seq"]
    hd, group, at = c["hd"], c["heads"] // c["kv"], 0
    out = torch.zeros_like(st["q"], dtype=torch.float64)
    for s, (n, total) in enumerate(zip(new, length)):
        if total and n:
            pages = st["table"][s, : -(-total // c["page"])].long()
            for h in range(c["heads"]):
                k, v = (x[pages, h // group].reshape(-1, hd)[:total].double() for x in (st["k_pages"], st["v_pages"]))
                score = st["q"][at:at + n, h * hd:(h + 1) * hd].double() @ k.T.contiguous() / hd ** 0.5
                if n > 1:
                    score.masked_fill_(torch.ones(n, total, dtype=torch.bool, device=DEV).triu_(total - n + 1), -math.inf)
                out[at:at + n, h * hd:(h + 1) * hd] = torch.softmax(score, -1) @ v
        at += n
    return out


def _exact_sample(st):
    x = st["logits"].double().cpu().numpy()
    t, k, p, low, u = (st[name].cpu().numpy() for name in ("temperature", "top_k", "top_p", "min_p", "u"))
    prob = np.empty(x.shape[0])
    for r in range(x.shape[0]):
        best = int(x[r].argmax())
        if t[r] <= 0 or k[r] == 1:
            prob[r] = 1.0
            continue
        order = np.argsort(-x[r], kind="stable")
        if k[r] > 0:
            order = order[: k[r]]
        w = np.exp((x[r, order] - x[r, best]) / float(t[r]))
        if 0 < p[r] < 1:
            order = order[: int(np.searchsorted(np.cumsum(w), float(p[r]) * w.sum(), side="left")) + 1]
        order = np.sort(order)
        w = np.exp((x[r, order] - x[r, best]) / float(t[r]))
        w = w[w >= float(low[r])]
        prob[r] = w[np.searchsorted(np.cumsum(w), u[r] * w.sum(), side="right").clip(max=w.size - 1)] / w.sum()
    return {"token": None, "prob": torch.from_numpy(prob)}


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    if case["op"] == "sample":
        return _exact_sample(st)
    return _exact_append(st) if case["op"] == "append" else _exact_attention(st)
