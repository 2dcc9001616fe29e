"""GPU: ie_sample against a plain 64-bit form."""
import math

import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


def run(ie, cuda, logits, u, **kw):
    M = logits.shape[0]
    idx = cuda.full((M,), -9, dtype=cuda.int32, device="cuda")
    logprob = cuda.full((M,), 9.0, device="cuda")
    ie.sample(logits, u, idx, logprob_out=logprob, **kw)
    cuda.cuda.synchronize()
    return idx, logprob


def check(ie, cuda, logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    idx, logprob = run(ie, cuda, logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    x = logits.double().cpu().tolist()
    get = lambda t, r, other: other if t is None else t[r].item()  # noqa: E731
    for r in range(len(x)):
        i, lp, margin = ref.sample_row(x[r], get(temperature, r, 1.0), get(top_k, r, 0), get(top_p, r, 1.0),
                                       get(min_p, r, 0.0), u[r].item())
        # masses agree to about 1e-15 relative a sum: a border nearer than 1e-12 is not told apart
        if margin > 1e-12:
            assert int(idx[r]) == i, (r, int(idx[r]), i)
            if lp == -math.inf:
                assert logprob[r].item() == lp
            else:  # one rounding to fp32 and the logarithm of 64-bit masses
                assert abs(logprob[r].item() - lp) <= 2.0 ** -24 * abs(lp) + 1e-12, (r, logprob[r].item(), lp)
    return idx


def inputs(cuda, M, V, dt, seed, std=3.0):
    g = cuda.Generator(device="cuda").manual_seed(seed)
    x = (std * cuda.randn((M, V), generator=g, device="cuda")).to(ref.DTYPES[dt])
    return x, cuda.rand(M, generator=g, device="cuda"), g


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("M,V", [(1, 1), (3, 2), (2, 7), (5, 8), (4, 9), (19, 1000), (40, 4097), (80, 1023),
                                 (160, 517), (2, 50257), (20, 128256), (1, 128256)])
def test_plain_temperature(ie, cuda, dt, M, V):
    x, u, g = inputs(cuda, M, V, dt, M + V)
    check(ie, cuda, x, u)
    check(ie, cuda, x, u, temperature=cuda.rand(M, generator=g, device="cuda") * 2 + 0.05)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("M,V", [(64, 300), (30, 5000), (8, 32001), (150, 999)])
def test_all_filters(ie, cuda, dt, M, V):
    x, u, g = inputs(cuda, M, V, dt, V)
    pick = lambda values, kind: cuda.tensor(values, dtype=kind, device="cuda")[  # noqa: E731
        cuda.randint(0, len(values), (M,), generator=g, device="cuda")]
    f32 = cuda.float32
    for _ in range(3):
        check(ie, cuda, x, u, temperature=pick([0.0, 0.3, 0.8, 1.0, 2.5], f32),
              top_k=pick([-1, 0, 1, 2, 5, 50, V - 1, V, V + 5], cuda.int32),
              top_p=pick([0.0, 0.1, 0.5, 0.9, 0.99, 1.0, 1.5], f32),
              min_p=pick([0.0, 0.01, 0.2, 1.0, -1.0], f32))


@pytest.mark.parametrize("top_k", [1, 3, 4, 10, 64])
@pytest.mark.parametrize("top_p", [0.3, 0.5, 0.75, 1.0])
def test_ties_go_to_the_lowest_id(ie, cuda, top_k, top_p):
    """Few distinct values: cuts fall inside a value, ranks inside it go by id."""
    M, V = 40, 1001
    g = cuda.Generator(device="cuda").manual_seed(top_k)
    x = cuda.randint(-2, 3, (M, V), generator=g, device="cuda").to(cuda.bfloat16)
    u = cuda.rand(M, generator=g, device="cuda")
    fill = lambda v, kind: cuda.full((M,), v, dtype=kind, device="cuda")  # noqa: E731
    check(ie, cuda, x, u, top_k=fill(top_k, cuda.int32), top_p=fill(top_p, cuda.float32))
    check(ie, cuda, x, u, top_p=fill(top_p, cuda.float32))


def test_equal_logits_and_counter_range(ie, cuda):
    """All logits equal: one counter takes a whole slice, and token floor(u V)
    is drawn; every u of a grid, the last token at u just below 1."""
    for V in (65528, 65529, 128256, 131056, 300001):
        x = cuda.zeros((3, V), dtype=cuda.float16, device="cuda")
        u = cuda.tensor([0.0, 0.5, 1 - 2.0 ** -24], device="cuda")
        idx, logprob = run(ie, cuda, x, u)
        assert idx.tolist() == [int(v * V) for v in u.tolist()]
        assert abs(logprob[0].item() + math.log(V)) <= 2.0 ** -23 * math.log(V)
    # one and two CTAs a row: slices close to a counter's largest value
    for V in (65504, 131000):
        x = cuda.zeros((75, V), dtype=cuda.float16, device="cuda")
        u = (cuda.arange(75, device="cuda") + 0.25) / 75
        idx, _ = run(ie, cuda, x, u)
        assert idx.tolist() == [int(v * V) for v in u.double().tolist()]


def test_signed_zero_nan_and_infinities(ie, cuda):
    inf, nan = math.inf, math.nan
    rows = [
        [-0.0, 0.0, -0.0, 0.0, -1.0, -1.0, -1.0, -1.0, -1.0],  # zeros are equal: ids 0 .. 3 in order
        [nan, -inf, 2.0, nan, 1.0, -inf, 1.0, nan, 0.0],
        [inf, 1.0, inf, -inf, nan, 5.0, 2.0, inf, 3.0],         # only the infinite ones
        [-inf] * 9, [nan] * 9, [nan, -inf] * 4 + [nan],
        [-inf] * 8 + [-60000.0],
        [65504.0, -65504.0] * 4 + [-65504.0],
        [1.0] * 9,
    ]
    for dt in ("f16", "bf16"):
        x = cuda.tensor(rows, device="cuda").to(ref.DTYPES[dt])
        for u in (0.0, 0.1, 0.34, 0.67, 0.999):
            for t in (1.0, 0.0, 1e-30, 1e30, inf, nan, -1.0):
                tt = cuda.full((len(rows),), t, device="cuda")
                if t == inf:
                    idx, _ = run(ie, cuda, x, cuda.full((len(rows),), u, device="cuda"), temperature=tt)
                    assert idx.tolist()[3:7] == [-1, -1, -1, 8]
                    continue
                check(ie, cuda, x, cuda.full((len(rows),), u, device="cuda"), temperature=tt)


def test_rows_and_strides(ie, cuda):
    """Rows of a wider buffer at odd element offsets; a row's neighbours hold
    larger logits that must not be seen."""
    V = 777
    for lead in range(9):
        big = cuda.full((6, V + 12), 60.0, dtype=cuda.float16, device="cuda")
        x, u, _ = inputs(cuda, 6, V, "f16", lead)
        big[:, lead:lead + V] = x
        got = check(ie, cuda, big[:, lead:lead + V], u)
        want, _ = run(ie, cuda, x, u)
        assert got.tolist() == want.tolist()


def test_u_at_the_ends(ie, cuda):
    x, _, _ = inputs(cuda, 4, 500, "bf16", 2)
    u = cuda.tensor([0.0, 1.0, 2.0, math.nan], device="cuda")
    k = cuda.full((4,), 10, dtype=cuda.int32, device="cuda")
    idx, _ = run(ie, cuda, x, u, top_k=k)
    order = cuda.sort(x.float(), dim=-1, descending=True, stable=True).indices
    assert idx.tolist() == [int(order[0, 0])] + [int(order[r, 9]) for r in (1, 2, 3)]


def test_parameters_outside_their_ranges(ie, cuda):
    """A negative u counts as 0; top_p of 0 or less, min_p above 1 and NaN of
    either keep the first token alone."""
    x, _, _ = inputs(cuda, 6, 500, "bf16", 2)
    first = cuda.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, 0].tolist()
    f = lambda *v: cuda.tensor(v, device="cuda")  # noqa: E731
    idx, lp = run(ie, cuda, x, f(-0.5, -0.0, -math.inf, -1e-30, 0.0, -2.0))
    assert idx.tolist() == first
    u = cuda.full((6,), 0.9, device="cuda")
    idx, lp = run(ie, cuda, x, u, top_p=f(0.0, -1.0, math.nan, 1e-30, 1.0, 1.0),
                  min_p=f(0.0, 0.0, 0.0, 0.0, 1.5, math.nan))
    assert idx.tolist() == first and lp.tolist() == [0.0] * 6


def test_a_row_does_not_depend_on_the_batch(ie, cuda):
    """1, 2, 4 and 8 CTAs a row give the same ids and log probabilities."""
    x, u, g = inputs(cuda, 160, 20011, "bf16", 3)
    p = cuda.full((160,), 0.9, device="cuda")
    idx, lp = run(ie, cuda, x, u, top_p=p)
    for n in (1, 18, 37, 74):
        a, b = run(ie, cuda, x[:n], u[:n], top_p=p[:n])
        assert a.tolist() == idx[:n].tolist()
        assert bool(((b - lp[:n]).abs() <= 2.0 ** -23 * lp[:n].abs()).all())


def test_distribution(ie, cuda):
    """A grid of u draws every kept token as often as its share says."""
    x = cuda.tensor([[2.0, 0.0, 1.0, -1.0, 1.0]], device="cuda").half()
    n = 4000
    u = (cuda.arange(n, device="cuda") + 0.5) / n
    idx, _ = run(ie, cuda, x.repeat(n, 1), u.float())
    share = cuda.softmax(x[0].double(), 0)
    count = cuda.bincount(idx.long(), minlength=5).double() / n
    assert bool(((count - share).abs() <= 1.0 / n + 1e-6).all())


def test_captured(ie, cuda):
    x, u, _ = inputs(cuda, 4, 3001, "bf16", 1)
    idx = cuda.zeros(4, dtype=cuda.int32, device="cuda")
    ie.sample(x, u, idx)
    cuda.cuda.synchronize()
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        ie.sample(x, u, idx)
    y, v, _ = inputs(cuda, 4, 3001, "bf16", 2)
    x.copy_(y)
    u.copy_(v)
    graph.replay()
    cuda.cuda.synchronize()
    assert idx.tolist() == run(ie, cuda, y, v)[0].tolist()
