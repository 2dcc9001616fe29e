"""GPU: paged attention where its arithmetic is strained: rows that one key
takes, weight spread over a long tail of small probabilities, equal values."""
import math

import pytest

import paged_bounds as pb
import paged_ref as ref
from test_gpu_paged import run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kind,q_lens,kv_lens", pb.PEAKED)
@pytest.mark.parametrize("q_factor,key_factor", [(1, 1), (8, 1), (40, 1), (40, 100)])
def test_peaked_scores(ie, cuda, dt, dim, kind, q_lens, kv_lens, q_factor, key_factor):
    s = pb.peaked_batch(q_lens, kv_lens, dt, q_factor, key_factor, dim=dim)
    want, bound = pb.attention(s, sum_of_rounded=kind == "few")
    assert bool(bound.isfinite().all())
    got = run_attention(ie, cuda, s)[:s["start"][-1]].double().reshape(want.shape)
    assert ie.device_status() == 0
    off = (got - want).abs()
    assert bool((off <= bound).all()), f"{float((off / bound).max())} of the bound"


def tail_batch(cuda, B, n, kv, gap, heads, kv_heads, dt, dim=64, page=64):
    """B sequences over the same pages. Key 0 scores `gap` and holds the value 0;
    all other keys score 0 and hold 1: a row at position p gives
    p / (p + e^gap)."""
    dtype = ref.DTYPES[dt]
    pages = -(-kv // page)
    e = lambda *shape, x=0.0: cuda.full(shape, x, dtype=dtype, device="cuda")  # noqa: E731
    k, v, q = e(pages, kv_heads, page, dim), e(pages, kv_heads, page, dim, x=1.0), e(B * n, heads, dim)
    k[0, :, 0, 0], v[0, :, 0], q[:, :, 0] = gap, 0.0, 1.0
    start = [n * b for b in range(B + 1)]
    table = cuda.arange(pages, dtype=cuda.int32, device="cuda").repeat(B, 1)
    return {"q": q, "k": k, "v": v, "table": table, "q_lens": [n] * B, "kv_lens": [kv] * B, "start": start,
            "page": page, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "q_start": cuda.tensor(start, dtype=cuda.int32, device="cuda"),
            "kv_len": cuda.full((B,), kv, dtype=cuda.int32, device="cuda")}


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("B,n,kv,heads,kv_heads", [
    (48, 1, 60000, 32, 8), (40, 4, 20001, 8, 8),     # few rows; enough sequences that a warp sees many keys
    (40, 64, 20000, 16, 8), (1, 700, 131071, 16, 4),  # chunks
])
@pytest.mark.parametrize("gap", [8.0, 12.0, 15.0, 16.0, 17.0, 17.5, 20.0])
def test_tail_of_small_probabilities(ie, cuda, dt, B, n, kv, heads, kv_heads, gap):
    """All of a long context beside one key that is e^gap times as likely. Every
    small p is rounded alike: u of the weight, or of the product only; the
    output's rounding u more; scores of at most 20 * 1.45 with 2^-24 twice, and
    2^-18 of the exponential, a tenth of fp16's u; and sums: a warp adds at most
    131071 / 16 times, where a step's rounding to even is at most 2^-24 of the
    sum so far, 2^-12 in all, on either sum. fp16 below its normal numbers: half
    a step, 2^-25, of the output, and of each p where the largest is at least
    2^7, so that kv of them are kv 2^-32 of the output's scale, 1."""
    s = tail_batch(cuda, B, n, kv, gap, heads, kv_heads, dt)
    got = run_attention(ie, cuda, s, scale=1.0).double().reshape(B, n, heads, s["dim"])
    assert ie.device_status() == 0
    p = cuda.arange(kv - n, kv, dtype=cuda.float64, device="cuda")[None, :, None, None]
    want = p / (p + math.exp(gap))
    bound = want * (3.1 * ref.half_step(ref.DTYPES[dt]) + 2 * 2.0 ** -12)
    if dt == "f16":
        bound = bound + 2.0 ** -25 + kv * 2.0 ** -32
    off = (got - want).abs()
    assert bool((off <= bound).all()), f"{float((off / bound).max())} of the bound"
