"""GPU: bounded waits of the paged attention kernels that do run out."""
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu

LIMITS = (1, 200, 400, 600, 800, 1000, 1500, 2000, 3000, 5000)  # ns: a copy from HBM takes about 1000


@pytest.mark.parametrize("dim,q_lens,kv_lens", [
    # few rows, in pieces and whole; at D = 64 only a batch that HBM bounds has to wait for its copies
    (128, [1, 1], [40000, 30000]), (128, [4], [100000]), (128, [1] * 64, [8000] * 64), (64, [4] * 64, [8000] * 64),
    # chunks
    (64, [200], [40000]), (128, [200], [40000]), (128, [700, 1], [9000, 20000]), (64, [30] * 40, [400] * 40),
])
def test_waits_run_out(ie, cuda, dim, q_lens, kv_lens):
    """Limits below the time that a copy takes make waits give up, the first
    ones or later ones: IE_ERR_TIMEOUT, the counters back at 0, nothing outside
    the output written, and the next call on the same workspace exact."""
    s = ref.make_batch(q_lens, kv_lens, dim=dim, seed=41, page=32)
    cache, ws = ie.PagedCache(s["k"], s["v"]), ie.paged_attention_workspace()
    ws[65536:].fill_(255)
    T = s["start"][-1]
    wide = cuda.full((T + 4, s["heads"] * s["dim"]), 5.0, dtype=s["q"].dtype, device="cuda")
    out = wide[2:2 + T]
    call = lambda: ie.paged_attention(s["q"], cache, s["table"], s["q_start"], s["kv_len"], out,  # noqa: E731
                                      max_q=max(q_lens), workspace=ws)
    flush = cuda.empty(1 << 28, dtype=cuda.uint8, device="cuda")
    want, bound = ref.attention(s)

    def exact():
        out.fill_(5.0)
        call()
        assert ie.device_status() == 0
        assert bool(((out.double().reshape(want.shape) - want).abs() <= bound).all())
        assert bool((wide[:2] == 5.0).all()) and bool((wide[2 + T:] == 5.0).all())

    ran_out = []
    try:
        for ns in LIMITS:
            ie.set_wait_limit_ns(ns)
            for _ in range(3):
                flush.fill_(1)  # the cache leaves L2
                call()
                status = ie.device_status()
                assert status in (0, -5)
                if status:
                    ran_out.append(ns)
                assert not bool(ws[:65536].any())
            ie.set_wait_limit_ns(0)
            exact()
    finally:
        ie.set_wait_limit_ns(0)
    assert LIMITS[0] in ran_out, ran_out


def test_a_limit_holds_until_the_next(ie, cuda):
    """A long limit after a short one: the waits are over in time again."""
    s = ref.make_batch([200], [40000], seed=42)
    cache, ws = ie.PagedCache(s["k"], s["v"]), ie.paged_attention_workspace()
    out = cuda.empty((s["start"][-1], s["heads"] * s["dim"]), dtype=s["q"].dtype, device="cuda")
    call = lambda: ie.paged_attention(s["q"], cache, s["table"], s["q_start"], s["kv_len"], out,  # noqa: E731
                                      max_q=200, workspace=ws)
    try:
        ie.set_wait_limit_ns(1)
        call()
        assert ie.device_status() == -5
        ie.set_wait_limit_ns(1_000_000_000)
        call()
        assert ie.device_status() == 0
    finally:
        ie.set_wait_limit_ns(0)
