"""GPU: the paged-cache operators and the sampler in a serving loop, as they
are used: projection, norm and rotation into pages, attention, projection,
sampling, with chunked prefill next to decoding sequences, pages handed out as
sequences grow, and decode steps replayed from a captured graph. Every stage is
checked against the 64-bit form of the inputs it had."""
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, H, V, PAGE = 8, 2, 64, 256, 1000, 16


class Loop:
    """One attention layer and a vocabulary projection over a paged cache."""

    def __init__(self, ie, cuda, slots, window=0, sinks=0, pages=64, wide=12):
        self.ie, self.cuda, self.window, self.sinks = ie, cuda, window, sinks
        g = cuda.Generator(device="cuda").manual_seed(5)
        draw = lambda *shape: (0.08 * cuda.randn(shape, generator=g, device="cuda")).bfloat16()  # noqa: E731
        self.emb, self.lm = (12 * draw(V, H)), draw(V, H) * 4
        self.wqkv, self.wo = draw((HEADS + 2 * KV_HEADS) * DIM, H), draw(H, HEADS * DIM)
        self.wq, self.wk = [(1 + draw(DIM)) for _ in range(2)]
        angle = cuda.arange(wide * PAGE, device="cuda", dtype=cuda.float64)[:, None] * \
            500000.0 ** (-cuda.arange(0, DIM, 2, device="cuda", dtype=cuda.float64) / DIM)
        self.cos, self.sin = angle.cos().float(), angle.sin().float()
        nan = lambda: cuda.full((pages, KV_HEADS, PAGE, DIM), float("nan"), dtype=cuda.bfloat16, device="cuda")  # noqa: E731
        self.k, self.v = nan(), nan()
        self.cache = ie.PagedCache(self.k, self.v)
        self.free = list(range(pages))[::-1]
        self.table = cuda.full((slots, wide), -1, dtype=cuda.int32, device="cuda")
        self.owned, self.length = [0] * slots, [0] * slots
        self.kv_len = cuda.zeros(slots, dtype=cuda.int32, device="cuda")
        self.q_start = cuda.zeros(slots + 1, dtype=cuda.int32, device="cuda")
        self.ws = ie.paged_attention_workspace()
        self.g = g

    def place(self, counts):
        """Room for counts[b] new tokens of each sequence; the device arrays follow."""
        for b, n in enumerate(counts):
            self.length[b] += n
            while self.owned[b] * PAGE < self.length[b]:
                self.table[b, self.owned[b]] = self.free.pop()
                self.owned[b] += 1
        self.kv_len.copy_(self.cuda.tensor(self.length, dtype=self.cuda.int32))
        start = [0]
        for n in counts:
            start.append(start[-1] + n)
        self.q_start.copy_(self.cuda.tensor(start, dtype=self.cuda.int32))
        return start

    def buffers(self, T, rows):
        e = lambda *shape, dt=self.cuda.bfloat16: self.cuda.zeros(shape, dtype=dt, device="cuda")  # noqa: E731
        return {"tokens": e(T, dt=self.cuda.int64), "x": e(T, H), "qkv": e(T, HEADS + 2 * KV_HEADS, DIM),
                "q": e(T, HEADS, DIM), "o": e(T, HEADS * DIM), "logits": e(rows, V), "u": e(rows, dt=self.cuda.float32),
                "ids": e(rows, dt=self.cuda.int32), "lp": e(rows, dt=self.cuda.float32),
                "t": self.cuda.full((rows,), 0.8, device="cuda"), "p": self.cuda.full((rows,), 0.9, device="cuda"),
                "k": self.cuda.full((rows,), 40, dtype=self.cuda.int32, device="cuda"),
                "last": e(rows, dt=self.cuda.int64)}

    def step(self, b, max_q):
        ie = self.ie
        b["x"].copy_(self.emb[b["tokens"]])
        ie.gemm(b["x"], self.wqkv, b["qkv"].view(len(b["x"]), -1))
        q, k, v = b["qkv"].split([HEADS, KV_HEADS, KV_HEADS], 1)
        ie.qk_norm_rope_paged(q, k, v, self.wq, self.wk, self.cos, self.sin, self.cache, self.table, self.q_start,
                              self.kv_len, b["q"])
        ie.paged_attention(b["q"], self.cache, self.table, self.q_start, self.kv_len, b["o"], max_q=max_q,
                           window=self.window, sinks=self.sinks, workspace=self.ws)
        ie.gemm_add(b["o"], self.wo, b["x"])
        ie.gemm(b["x"][b["last"]], self.lm, b["logits"])
        ie.sample(b["logits"], b["u"], b["ids"], temperature=b["t"], top_k=b["k"], top_p=b["p"], logprob_out=b["lp"])

    def check(self, b, counts, start):
        cuda = self.cuda
        assert self.ie.device_status() == 0
        n = start[-1]
        # attention, from the cache as it stands
        s = {"q": b["q"][:n], "k": self.k, "v": self.v, "table": self.table, "q_lens": counts,
             "kv_lens": self.length, "start": start, "page": PAGE, "heads": HEADS, "kv_heads": KV_HEADS, "dim": DIM}
        want, bound = ref.attention(s, self.window, self.sinks)
        assert bool(((b["o"][:n].double().reshape(want.shape) - want).abs() <= bound).all())
        for i, m in enumerate(counts):
            if not m:
                continue
            t = slice(start[i], start[i] + m)
            pos = cuda.arange(self.length[i] - m, self.length[i], device="cuda")
            u = ref.half_step(cuda.bfloat16)
            for got, part, w in ((b["q"][t], b["qkv"][t, :HEADS], self.wq),
                                 (self.k[self.table[i].long()[pos // PAGE], :, pos % PAGE],
                                  b["qkv"][t, HEADS:HEADS + KV_HEADS], self.wk)):
                y = ref.norm_rope(part, w, self.cos, self.sin, pos, 1e-5)
                mag = y.abs().amax(-1, keepdim=True) * 2
                assert bool(((got.double() - y).abs() <= u * y.abs() + (DIM + 16) * 2.0 ** -24 * mag).all())
            assert bool((self.v[self.table[i].long()[pos // PAGE], :, pos % PAGE] ==
                         b["qkv"][t, HEADS + KV_HEADS:]).all())
        logits = b["logits"].double().cpu().tolist()
        for r, x in enumerate(logits):
            i, lp, margin = ref.sample_row(x, b["t"][r].item(), 40, b["p"][r].item(), 0.0, b["u"][r].item())
            if margin > 1e-12:
                assert int(b["ids"][r]) == i and abs(b["lp"][r].item() - lp) <= 2.0 ** -24 * abs(lp) + 1e-12


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
def test_serving_loop(ie, cuda, window, sinks):
    loop = Loop(ie, cuda, 3, window, sinks)
    rand = lambda n: cuda.randint(0, V, (n,), generator=loop.g, device="cuda")  # noqa: E731
    # chunked prefill: 70 tokens of sequence 0 in two chunks, 5 of sequence 1
    # with the first, one decode step of sequence 1 next to the second
    for counts in ([48, 5, 0], [22, 1, 0], [0, 1, 33]):
        start = loop.place(counts)
        T, rows = start[-1] + 2, 3
        b = loop.buffers(T, rows)
        b["tokens"].copy_(rand(T))
        b["u"].copy_(cuda.rand(rows, generator=loop.g, device="cuda"))
        b["last"].copy_(cuda.tensor([max(start[i + 1] - 1, 0) for i in range(3)]))
        b["o"].fill_(0)
        loop.step(b, max(counts))
        loop.check(b, counts, start)
    # decode: one captured step, replayed as the sequences grow over page ends
    b = loop.buffers(3, 3)
    b["last"].copy_(cuda.arange(3))
    side = cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    start = loop.place([1, 1, 1])
    b["tokens"].copy_(rand(3))
    with cuda.cuda.stream(side):
        loop.step(b, 1)
    side.synchronize()
    loop.check(b, [1, 1, 1], start)
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        loop.step(b, 1)
    for _ in range(20):
        start = loop.place([1, 1, 1])
        b["tokens"].copy_(b["ids"].long())
        b["u"].copy_(cuda.rand(3, generator=loop.g, device="cuda"))
        graph.replay()
        loop.check(b, [1, 1, 1], start)
    # a sequence leaves: its slot is empty, the others go on
    loop.length[1] = 0
    start = loop.place([1, 0, 1])
    b["o"].fill_(9.0)
    graph.replay()
    loop.check(b, [1, 0, 1], start)
    assert bool((b["o"][2] == 9.0).all())


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [900, 3000]), ([200], [3000]), ([64], [9000]), ([2100], [2100])])
def test_a_wait_that_runs_out_leaves_the_context_usable(ie, cuda, q_lens, kv_lens):
    """With a limit of 1 ns a wait for a copy may run out: the call then records
    IE_ERR_TIMEOUT and ends, and the next call on the same workspace is exact."""
    s = ref.make_batch(q_lens, kv_lens, seed=3, page=32)
    cache, ws = ie.PagedCache(s["k"], s["v"]), ie.paged_attention_workspace()
    ws[65536:].fill_(255)
    out = cuda.empty((s["start"][-1], s["heads"] * s["dim"]), dtype=s["q"].dtype, device="cuda")
    call = lambda: ie.paged_attention(s["q"], cache, s["table"], s["q_start"], s["kv_len"], out,  # noqa: E731
                                      max_q=max(q_lens), workspace=ws)
    try:
        ie.set_wait_limit_ns(1)
        for _ in range(3):
            call()
            assert ie.device_status() in (0, -5)
    finally:
        ie.set_wait_limit_ns(0)
    call()
    assert ie.device_status() == 0
    want, bound = ref.attention(s)
    assert bool(((out.double().reshape(want.shape) - want).abs() <= bound).all())
    assert not bool(ws[:65536].any())
