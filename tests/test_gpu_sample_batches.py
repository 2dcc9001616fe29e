"""GPU: ie_sample over every batch size around which its CTAs a row change."""
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


def test_fewer_rows_do_not_take_longer(ie, cuda):
    """CTAs a row are chosen so that a batch runs at once: no batch takes much
    longer than a larger one does. Best of 9 replays of 8 calls; a second wave
    of clusters made it 1.7 times as long."""
    V, most = 32001, 80
    x = cuda.randn((most, V), device="cuda").half()
    u, idx = cuda.rand(most, device="cuda"), cuda.zeros(most, dtype=cuda.int32, device="cuda")
    graphs = []
    for M in range(1, most + 1):
        ie.sample(x[:M], u[:M], idx[:M])
        cuda.cuda.synchronize()
        graphs.append(cuda.cuda.CUDAGraph())
        with cuda.cuda.graph(graphs[-1]):
            for _ in range(8):
                ie.sample(x[:M], u[:M], idx[:M])
    best = [float("inf")] * most
    a, b = [cuda.cuda.Event(enable_timing=True) for _ in range(2)]
    for _ in range(9):
        for i, g in enumerate(graphs):
            a.record()
            g.replay()
            b.record()
            cuda.cuda.synchronize()
            best[i] = min(best[i], a.elapsed_time(b))
    for i in range(most - 1):
        assert best[i] <= 1.4 * min(best[i + 1:]), (i + 1, best)


@pytest.mark.parametrize("dt,V", [("f16", 20011), ("bf16", 128256)])
def test_rows_are_the_same_in_every_batch(ie, cuda, dt, V):
    g = cuda.Generator(device="cuda").manual_seed(V)
    x = (3 * cuda.randn((80, V), generator=g, device="cuda")).to(ref.DTYPES[dt])
    u, p = cuda.rand(80, generator=g, device="cuda"), cuda.full((80,), 0.9, device="cuda")
    idx, lp = cuda.zeros(80, dtype=cuda.int32, device="cuda"), cuda.zeros(80, device="cuda")
    ie.sample(x, u, idx, top_p=p, logprob_out=lp)
    for M in (1, 14, 15, 16, 17, 18, 19, 32, 33, 34, 36, 37, 38, 73, 74, 75):
        i, l = cuda.zeros_like(idx[:M]), cuda.zeros_like(lp[:M])
        ie.sample(x[:M], u[:M], i, top_p=p[:M], logprob_out=l)
        assert i.tolist() == idx[:M].tolist()
        # masses of another order of summation: one step of the 32-bit logarithm
        assert bool(((l - lp[:M]).abs() <= 2.0 ** -23 * lp[:M].abs()).all())
