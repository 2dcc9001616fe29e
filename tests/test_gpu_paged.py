"""GPU: the paged-cache operators (attention, norm + rotation + page write)
against plain 64-bit forms."""
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


def run_attention(ie, cuda, s, window=0, sinks=0, scale=None, out=None, max_q=None, workspace=None, **kw):
    cache = ie.PagedCache(s["k"], s["v"])
    T = s["q"].shape[0]
    if out is None:
        out = cuda.full((T, s["heads"] * s["dim"]), 77.0, dtype=s["q"].dtype, device="cuda")
    if workspace is None:
        workspace = ie.paged_attention_workspace()
        workspace[65536:].fill_(255)  # whatever it holds behind the counters: NaN as floats
    ie.paged_attention(s["q"], cache, s["table"], s["q_start"], s["kv_len"], out,
                       max_q=max(s["q_lens"] + [0]) if max_q is None else max_q, window=window, sinks=sinks,
                       scale=scale, workspace=workspace, **kw)
    assert not bool(workspace[:65536].any())  # the counters are back at 0
    return out


def check_attention(ie, cuda, s, window=0, sinks=0, scale=None, **kw):
    out = run_attention(ie, cuda, s, window, sinks, scale, **kw)
    assert ie.device_status() == 0
    want, bound = ref.attention(s, window, sinks, scale)
    n = s["start"][-1]
    got = out[:n].double().reshape(want.shape)
    assert not got.isnan().any()
    off = (got - want).abs()
    assert bool((off <= bound).all()), f"{float((off / bound).max())} of the bound"
    assert bool((out[n:] == 77.0).all())  # rows no sequence owns
    return out


LENGTHS = [
    ([1], [1]), ([1], [2]), ([1], [15]), ([1], [16]), ([1], [17]), ([1], [31]), ([1], [33]), ([1], [127]),
    ([1], [129]), ([1], [1000]), ([1], [5003]),
    ([1, 1, 1, 1, 1], [1, 70, 300, 2049, 16]),
    ([2], [2]), ([3], [40]), ([5, 5], [5, 261]), ([4, 1, 0, 2], [100, 1, 50, 33]),
    ([0, 0], [10, 0]), ([1, 0, 1], [20, 0, 64]), ([1, 1], [0, 9]),
    ([7], [3]),   # four rows before the first cached one see nothing
]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("q_lens,kv_lens", LENGTHS)
def test_attention_few_rows(ie, cuda, dt, q_lens, kv_lens):
    check_attention(ie, cuda, ref.make_batch(q_lens, kv_lens, dt=dt, seed=len(kv_lens) + kv_lens[0], spare_rows=3))


CHUNKS = [
    ([16], [16]), ([17], [17]), ([64], [64]), ([65], [200]), ([100], [1000]), ([128], [128]), ([129], [129]),
    ([255], [300]), ([256], [256]), ([257], [700]), ([300, 1, 0, 33], [300, 900, 20, 64]), ([1, 500], [2000, 511]),
    ([40], [11]),
    ([2100], [2100]), ([900, 1500], [3500, 1501]),  # more tiles than SMs: whole ranges of many blocks
]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("q_lens,kv_lens", CHUNKS)
def test_attention_chunks(ie, cuda, dt, q_lens, kv_lens):
    heads = 8 if max(q_lens) < 900 else 20
    check_attention(ie, cuda, ref.make_batch(q_lens, kv_lens, heads=heads, kv_heads=heads // 4, dt=dt,
                                             seed=q_lens[0], spare_rows=5))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (6, 2), (5, 5), (8, 1), (16, 1), (14, 2), (32, 8)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [3, 200, 1111]), ([6, 1], [90, 70]), ([130, 20], [400, 20])])
def test_attention_head_layouts(ie, cuda, heads, kv_heads, dim, q_lens, kv_lens):
    check_attention(ie, cuda, ref.make_batch(q_lens, kv_lens, heads=heads, kv_heads=kv_heads, dim=dim, seed=heads))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["hnd", "nhd", "padded"])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [77, 1025]), ([70, 3], [333, 40])])
def test_attention_pages_and_orders(ie, cuda, page, layout, q_lens, kv_lens):
    check_attention(ie, cuda, ref.make_batch(q_lens, kv_lens, page=page, layout=layout, dt="f16", seed=page))


WINDOWS = [(1, 0), (2, 1), (16, 0), (16, 4), (33, 17), (64, 100), (100, 5), (1000, 4), (5000, 4)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [1, 90, 777]), ([5], [130]), ([200, 30], [700, 31])])
def test_attention_window(ie, cuda, window, sinks, page, q_lens, kv_lens):
    s = ref.make_batch(q_lens, kv_lens, page=page, seed=window + sinks)
    # pages and rows that no row sees hold NaN, and their table entries lead nowhere
    for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        first = max(0, kv - n - window + 1)
        for j in range(min(sinks, first), first):
            s["k"][int(s["table"][b, j // page]), :, j % page] = float("nan")
            s["v"][int(s["table"][b, j // page]), :, j % page] = float("nan")
    want = check_attention(ie, cuda, s, window, sinks)
    for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        first = max(0, kv - n - window + 1)
        for i in range(-(-min(sinks, first) // page), first // page):
            s["table"][b, i] = -1 if i % 2 else 1 << 30
    got = run_attention(ie, cuda, s, window, sinks)
    assert ie.device_status() == 0
    assert bool((got == want).all())


@pytest.mark.parametrize("q_lens,kv_lens", [([1], [300]), ([80], [300])])
@pytest.mark.parametrize("scale", [0.0, 1.0, -0.1, 0.3])
def test_attention_scale(ie, cuda, q_lens, kv_lens, scale):
    check_attention(ie, cuda, ref.make_batch(q_lens, kv_lens, dt="f16", seed=4), scale=scale)


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [900, 80]), ([90, 2], [300, 40])])
def test_attention_extreme_scores(ie, cuda, q_lens, kv_lens):
    """Scores of the type's largest values on either side: one key takes all,
    and a whole row far below the others' exponent range."""
    s = ref.make_batch(q_lens, kv_lens, dt="bf16", seed=8)
    s["q"].mul_(40.0)
    check_attention(ie, cuda, s)
    s["k"][int(s["table"][0, 0]), :, 3] *= 100
    check_attention(ie, cuda, s)


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [50, 300, 7]), ([3], [90]), ([150, 1], [300, 17])])
def test_attention_strides(ie, cuda, q_lens, kv_lens):
    """Queries head-major and as columns of a wider projection, an output that
    is part of a wider buffer."""
    s = ref.make_batch(q_lens, kv_lens, seed=5)
    want = check_attention(ie, cuda, s)
    T, heads, dim = s["q"].shape
    fused = cuda.full((T, heads + 4, dim), float("nan"), dtype=s["q"].dtype, device="cuda")
    fused[:, 2:2 + heads] = s["q"]
    wide = cuda.full((T, heads * dim + 64), 3.0, dtype=s["q"].dtype, device="cuda")
    for q in (s["q"].transpose(0, 1).contiguous().transpose(0, 1), fused[:, 2:2 + heads]):
        got = run_attention(ie, cuda, dict(s, q=q), out=wide[:, 8:8 + heads * dim])
        assert bool((got == want).all())
    assert bool((wide[:, :8] == 3.0).all()) and bool((wide[:, 8 + heads * dim:] == 3.0).all())


def test_attention_offsets_past_32_bits(ie, cuda):
    """Pages whose elements lie further than 2^32 from the pool's start."""
    dim, page, kv_heads = 128, 16, 2
    s = ref.make_batch([1, 40], [100, 70], dim=dim, page=page, kv_heads=kv_heads, heads=8, seed=6)
    pages = (1 << 32) // (dim * page * kv_heads) + 64
    first = pages - s["k"].shape[0]
    for x in ("k", "v"):
        big = cuda.empty((pages, kv_heads, page, dim), dtype=s["q"].dtype, device="cuda")
        big[first:] = s[x]
        s[x] = big
    s["table"] = cuda.where(s["table"] >= 0, s["table"] + first, s["table"])
    check_attention(ie, cuda, s)


def test_attention_bits_and_long_context(ie, cuda):
    """The same call gives the same bits; a long context is cut over the GPU."""
    for q_lens, kv_lens in (([1], [40000]), ([5, 1], [9000, 30000]), ([64], [20000]), ([300], [9000])):
        s = ref.make_batch(q_lens, kv_lens, heads=8, kv_heads=2, dt="f16", page=64, seed=9)
        a = check_attention(ie, cuda, s)
        for _ in range(3):
            assert bool((run_attention(ie, cuda, s) == a).all())


@pytest.mark.parametrize("max_q", [1, 48])
def test_attention_captured(ie, cuda, max_q):
    """A captured call follows the lengths, the table and the contents; a
    sequence slot may be empty."""
    s = ref.make_batch([max_q, max_q, max_q], [1000, 900, 800], seed=10, page=32)
    cache = ie.PagedCache(s["k"], s["v"])
    ws = ie.paged_attention_workspace()
    out = cuda.zeros((3 * max_q, s["heads"] * s["dim"]), dtype=s["q"].dtype, device="cuda")
    call = lambda: ie.paged_attention(s["q"], cache, s["table"], s["q_start"], s["kv_len"], out, max_q=max_q,  # noqa: E731
                                      workspace=ws)
    call()
    cuda.cuda.synchronize()
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        call()
    for q_lens, kv_lens in (([max_q, 0, 1], [700, 0, 33]), ([1, max_q, 0], [1, 555, 10])):
        new = dict(s, q_lens=q_lens, kv_lens=kv_lens, start=[0, q_lens[0], q_lens[0] + q_lens[1], sum(q_lens)])
        s["q_start"].copy_(cuda.tensor(new["start"], dtype=cuda.int32))
        s["kv_len"].copy_(cuda.tensor(kv_lens, dtype=cuda.int32))
        out.fill_(77.0)
        graph.replay()
        assert ie.device_status() == 0
        want, bound = ref.attention(new)
        n = new["start"][-1]
        assert bool(((out[:n].double().reshape(want.shape) - want).abs() <= bound).all())
        assert bool((out[n:] == 77.0).all())


def test_attention_other_stream(ie, cuda):
    s = ref.make_batch([1, 20], [500, 60], seed=11)
    want = check_attention(ie, cuda, s)
    side = cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    got = run_attention(ie, cuda, s, stream=side)
    side.synchronize()
    assert bool((got == want).all())
    with cuda.cuda.stream(side):
        got = run_attention(ie, cuda, s)
    side.synchronize()
    assert bool((got == want).all())


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [60, 40]), ([30, 20], [60, 40])])
def test_attention_bad_extents_set_the_status(ie, cuda, q_lens, kv_lens):
    """A page outside the pool, a length past the table, more new tokens than
    max_q: no access, IE_ERR_INVALID_ARG, and the other sequence is exact."""
    good = ref.make_batch(q_lens, kv_lens, seed=12)
    want, bound = ref.attention(good)
    n0 = q_lens[0]

    def bad_call(**change):
        s = dict(good, table=good["table"].clone(), kv_len=good["kv_len"].clone())
        max_q = None
        if "page" in change:
            s["table"][1, 1] = change["page"]
        if "kv" in change:
            s["kv_len"][1] = change["kv"]
        if "max_q" in change:
            max_q = change["max_q"]
        out = run_attention(ie, cuda, s, max_q=max_q)
        assert ie.device_status() == -1
        assert ie.device_status() == 0
        return out

    for change in ({"page": 1 << 30}, {"page": -1}, {"page": s_pages(good)}, {"kv": 1 << 30}, {"kv": -5}):
        out = bad_call(**change)
        got = out[:n0].double().reshape(n0, good["heads"], good["dim"])
        assert bool(((got - want[:n0]).abs() <= bound[:n0]).all())
    if q_lens[0] > 1:
        bad_call(max_q=q_lens[0] - 1)


def s_pages(s):
    return s["k"].shape[0]


# ------------------------------------------------------------- norm + rotation
def run_norm(ie, cuda, dt, q_lens, kv_lens, heads, kv_heads, dim, page, layout="hnd", weights=True, rope=True,
             order="fused", in_place=False, spare=0, seed=0):
    s = ref.make_batch(q_lens, kv_lens, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dt=dt, layout=layout,
                       seed=seed, spare_rows=spare)
    g = cuda.Generator(device="cuda").manual_seed(seed + 1)
    dtype = ref.DTYPES[dt]
    T = s["q"].shape[0]
    x = (2 * cuda.randn((T, heads + 2 * kv_heads, dim), generator=g, device="cuda")).to(dtype)
    if order == "head":
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    wq = wk = None
    if weights:
        wq, wk = [(1 + 0.3 * cuda.randn(dim, generator=g, device="cuda")).to(dtype) for _ in range(2)]
    cos = sin = None
    if rope:
        top = max(kv_lens + [1])
        angle = cuda.arange(top, device="cuda", dtype=cuda.float64)[:, None] * \
            500000.0 ** (-cuda.arange(0, dim, 2, device="cuda", dtype=cuda.float64) / dim)
        cos, sin = angle.cos().float(), angle.sin().float()
    cache = ie.PagedCache(s["k"], s["v"])
    k_before, v_before = s["k"].clone(), s["v"].clone()
    q_in = q.clone()
    out = q if in_place else cuda.full((T, heads, dim), 77.0, dtype=dtype, device="cuda")
    ie.qk_norm_rope_paged(q, k, v, wq, wk, cos, sin, cache, s["table"], s["q_start"], s["kv_len"], out, eps=1e-5)
    assert ie.device_status() == 0
    u = ref.half_step(dtype)

    def close(got, want, mag):
        # one rounding, and fp32: a norm of dim terms, two products and a sum
        bound = u * want.abs() + (dim + 16) * 2.0 ** -24 * mag + \
            cuda.finfo(dtype).smallest_normal * cuda.finfo(dtype).eps
        assert bool(((got.double() - want).abs() <= bound).all())

    want_k, want_v = k_before, v_before
    for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        t = slice(s["start"][b], s["start"][b] + n)
        pos = cuda.arange(kv - n, kv, device="cuda")
        full = lambda x, w: ref.norm_rope(x, w, cos, sin, pos, 1e-5)  # noqa: E731
        mag = lambda x, w: ref.norm_rope(x, w, None, None, pos, 1e-5).abs().amax(-1, keepdim=True) * 2  # noqa: E731
        close(out[t], full(q_in[t], wq), mag(q_in[t], wq))
        at, row = s["table"][b].long()[pos // page], pos % page
        close(s["k"][at, :, row], full(k[t], wk), mag(k[t], wk))
        assert bool((s["v"][at, :, row] == v[t]).all())
        want_k[at, :, row] = s["k"][at, :, row]
        want_v[at, :, row] = s["v"][at, :, row]
    # nothing else of the cache, and no row that no sequence owns, was touched
    assert bool(((s["k"] == want_k) | (s["k"].isnan() & want_k.isnan())).all())
    assert bool(((s["v"] == want_v) | (s["v"].isnan() & want_v.isnan())).all())
    rest = out[s["start"][-1]:]
    assert bool((rest == (q_in[s["start"][-1]:] if in_place else 77.0)).all())


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_lens,kv_lens", [([1], [1]), ([1, 1, 1], [5, 17, 300]), ([0, 3, 0, 1], [4, 3, 0, 16]),
                                            ([33, 1, 100], [50, 2000, 100])])
def test_norm_rope(ie, cuda, dt, dim, q_lens, kv_lens):
    run_norm(ie, cuda, dt, q_lens, kv_lens, 8, 2, dim, 16, spare=2)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (7, 7), (32, 8), (9, 3)])
@pytest.mark.parametrize("layout,order,in_place,page", [("nhd", "fused", False, 32), ("padded", "head", False, 64),
                                                        ("hnd", "fused", True, 16), ("hnd", "head", True, 256)])
def test_norm_rope_layouts(ie, cuda, heads, kv_heads, layout, order, in_place, page):
    run_norm(ie, cuda, "bf16", [2, 70, 1], [40, 300, 9], heads, kv_heads, 128, page, layout=layout, order=order,
             in_place=in_place, spare=1, seed=heads)


@pytest.mark.parametrize("weights,rope", [(False, True), (True, False), (False, False)])
def test_norm_rope_parts(ie, cuda, weights, rope):
    run_norm(ie, cuda, "f16", [3, 1], [30, 20], 4, 2, 64, 16, weights=weights, rope=rope)


def test_norm_rope_many_sequences(ie, cuda):
    """Owners by search: more sequences than a warp has lanes, empty ones among them."""
    q_lens = [(b * 7) % 4 for b in range(1100)]
    run_norm(ie, cuda, "bf16", q_lens, [n + b % 50 for b, n in enumerate(q_lens)], 2, 1, 64, 16, spare=4)


def test_norm_rope_large(ie, cuda):
    run_norm(ie, cuda, "bf16", [1500, 900], [2000, 901], 32, 8, 128, 64, spare=1)


def test_norm_rope_bad_extents_set_the_status(ie, cuda):
    """A page outside the pool and a position without a rotation row: that
    token is skipped, the others are written."""
    s = ref.make_batch([1, 1, 1], [20, 40, 60], heads=2, kv_heads=1, dim=64, seed=3)
    x = cuda.randn((3, 4, 64), device="cuda").bfloat16()
    s["table"][0, 1] = s["k"].shape[0]
    cos, sin = cuda.ones((50, 32), device="cuda"), cuda.zeros((50, 32), device="cuda")
    out = cuda.full((3, 2, 64), 77.0, dtype=cuda.bfloat16, device="cuda")
    ie.qk_norm_rope_paged(x[:, :2], x[:, 2:3], x[:, 3:], None, None, cos, sin, ie.PagedCache(s["k"], s["v"]),
                          s["table"], s["q_start"], s["kv_len"], out)
    assert ie.device_status() == -1
    assert bool((out[0] == 77.0).all()) and bool((out[2] == 77.0).all()) and bool((out[1] == x[1, :2]).all())
    at = int(s["table"][1, 39 // 16])
    assert bool((s["v"][at, 0, 39 % 16] == x[1, 3]).all())


# -------------------------------------------------- batches of other shapes
def many(B, longest, most_new, seed):
    """B sequences of 0 .. most_new new tokens, one of them far longer than the others."""
    g = __import__("random").Random(seed)
    q_lens = [g.choice([0, 1, 1, most_new, g.randint(1, most_new)]) for _ in range(B)]
    kv_lens = [n + g.randint(0, 150) for n in q_lens]
    q_lens[B // 2], kv_lens[B // 2] = most_new, longest
    return q_lens, kv_lens


@pytest.mark.parametrize("B", [32, 33, 64, 150, 300])
@pytest.mark.parametrize("most_new,longest", [(1, 6000), (6, 900), (40, 5000)])
def test_attention_many_sequences(ie, cuda, B, most_new, longest):
    q_lens, kv_lens = many(B, longest, most_new, B + most_new)
    check_attention(ie, cuda, ref.make_batch(q_lens, kv_lens, heads=4, kv_heads=1, dim=64, page=32, seed=B))
    if most_new == 6:
        check_attention(ie, cuda, ref.make_batch(q_lens, kv_lens, heads=4, kv_heads=1, dim=64, page=32, seed=B),
                        window=40, sinks=3)


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [60, 300]), ([50, 3], [60, 400])])
def test_attention_rows_outside_the_batch(ie, cuda, q_lens, kv_lens):
    """Rows before the first and behind the last sequence hold NaN: they are
    neither written nor felt."""
    s = ref.make_batch(q_lens, kv_lens, seed=21)
    want = check_attention(ie, cuda, s)
    T, heads, dim = s["q"].shape
    q = cuda.full((T + 9, heads, dim), float("nan"), dtype=s["q"].dtype, device="cuda")
    q[4:4 + T] = s["q"]
    out = run_attention(ie, cuda, dict(s, q=q, q_start=s["q_start"] + 4))
    assert ie.device_status() == 0
    assert bool((out[4:4 + T] == want).all())
    assert bool((out[:4] == 77.0).all()) and bool((out[4 + T:] == 77.0).all())


@pytest.mark.parametrize("n", [1, 30])
def test_attention_shared_pages(ie, cuda, n):
    """Sequences that begin with the same pages, and one listed twice."""
    s = ref.make_batch([n, n, n], [200, 230, 200], seed=22)
    s["table"][1, :8] = s["table"][0, :8]
    s["table"][2] = s["table"][0]
    out = check_attention(ie, cuda, s)
    s["q"][2 * n:] = s["q"][:n]
    out = check_attention(ie, cuda, s)
    assert bool((out[2 * n:] == out[:n]).all())


def test_attention_two_calls_at_once(ie, cuda):
    """Two streams, a workspace each: both as they are alone."""
    batches = [ref.make_batch([1], [30000], dim=64, page=64, seed=23), ref.make_batch([70], [9000], page=64, seed=24),
               ref.make_batch([2, 1], [7000, 50], page=64, seed=25)]
    want = [check_attention(ie, cuda, s) for s in batches]
    streams = [cuda.cuda.Stream() for _ in batches]
    ws = [ie.paged_attention_workspace() for _ in batches]
    caches = [ie.PagedCache(s["k"], s["v"]) for s in batches]
    outs = [[cuda.zeros_like(w) for _ in range(6)] for w in want]
    cuda.cuda.synchronize()
    for x in range(6):
        for s, c, o, w, st in zip(batches, caches, outs, ws, streams):
            ie.paged_attention(s["q"], c, s["table"], s["q_start"], s["kv_len"], o[x], max_q=max(s["q_lens"]),
                               workspace=w, stream=st)
    cuda.cuda.synchronize()
    assert ie.device_status() == 0
    for o, w in zip(outs, want):
        assert all(bool((y == w).all()) for y in o)


@pytest.mark.parametrize("B", [3, 40])
@pytest.mark.parametrize("n", [4, 40])
def test_attention_starts_that_decrease(ie, cuda, B, n):
    """Starts out of order are reported; counters and later calls stay sound."""
    s = ref.make_batch([n] * B, [900] * B, heads=4, kv_heads=1, dim=64, page=64, seed=26)
    want = check_attention(ie, cuda, s)
    start = s["q_start"].clone()
    start[1::2] = 0
    run_attention(ie, cuda, dict(s, q_start=start))
    assert ie.device_status() == -1
    run_attention(ie, cuda, dict(s, q_start=start.flip(0) - n))
    assert ie.device_status() == -1
    assert bool((check_attention(ie, cuda, s) == want).all())


def test_attention_workspace_refusals(ie, cuda):
    s = ref.make_batch([1], [9], seed=27)
    n = ie.paged_attention_workspace_bytes()
    with pytest.raises(ie.IEError):
        run_attention(ie, cuda, s, workspace=cuda.zeros(n - 1, dtype=cuda.uint8, device="cuda"))
    with pytest.raises(ValueError, match="contiguous"):
        run_attention(ie, cuda, s, workspace=cuda.zeros(16, dtype=cuda.uint8, device="cuda")[:1].expand(n))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (8, 2, 64), (16, 1, 128), (6, 2, 64)])
@pytest.mark.parametrize("kv_lens", [
    [448, 449, 512, 300, 513],       # from 8 blocks of 64 keys on a few rows' blocks are shared out
    [576, 577, 9000, 300, 20000],    # odd numbers of blocks, and cut tiles
])
@pytest.mark.parametrize("window,sinks", [(0, 0), (530, 70), (100, 3)])
def test_attention_few_rows_beside_a_chunk(ie, cuda, dt, heads, kv_heads, dim, kv_lens, window, sinks):
    """Sequences of one to a few tokens in a batch with a chunk."""
    few = 32 // (heads // kv_heads)
    s = ref.make_batch([1, 2, few, 150, few + 1], kv_lens, heads=heads, kv_heads=kv_heads, dim=dim, dt=dt, page=32,
                       seed=31)
    a = check_attention(ie, cuda, s, window=window, sinks=sinks)
    assert bool((run_attention(ie, cuda, s, window=window, sinks=sinks) == a).all())


def test_attention_many_single_tokens_beside_a_chunk(ie, cuda):
    """More pieces that both lanes serve than CTAs, next to others."""
    kv_lens = [600 + 37 * b for b in range(30)] + [900]
    check_attention(ie, cuda, ref.make_batch([1] * 30 + [300], kv_lens, heads=32, kv_heads=8, page=64, seed=32))
    kv_lens = [500 + 19 * b for b in range(60)] + [900, 2000]
    check_attention(ie, cuda, ref.make_batch([1, 2] * 30 + [300, 60], kv_lens, heads=16, kv_heads=4, dim=64, seed=33))


@pytest.mark.parametrize("B", [31, 32])
def test_attention_verification_batches(ie, cuda, B):
    """Five tokens a sequence, on both sides of the rule that picks the kernel."""
    q_lens = [5 - b % 3 for b in range(B)]
    check_attention(ie, cuda, ref.make_batch(q_lens, [5 + (b * 97) % 1300 for b in range(B)], seed=34))


@pytest.mark.parametrize("q_lens,kv_lens", [([0, 1, 3], [9000, 40, 700]), ([0, 90, 1], [9000, 500, 700])])
def test_attention_long_sequence_without_new_tokens(ie, cuda, q_lens, kv_lens):
    """A slot that keeps its length but brings no rows does not change the others' bits."""
    s = ref.make_batch(q_lens, kv_lens, seed=35)
    a = check_attention(ie, cuda, s)
    s["kv_len"][0] = 0
    assert bool((run_attention(ie, cuda, s) == a).all())
