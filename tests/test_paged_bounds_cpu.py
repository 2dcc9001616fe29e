"""CPU: the error bound of the paged attention tests holds for the plain
arithmetic it stands for, and is narrow enough to notice wrong outputs."""
import pytest
import torch

import paged_bounds as pb
import paged_ref as ref


def emulate(s, sum_of_rounded):
    """The operator with fp32 scores and sums, p and the output rounded to the type."""
    dtype, group = s["q"].dtype, s["heads"] // s["kv_heads"]
    out = torch.zeros((s["start"][-1], s["heads"], s["dim"]), dtype=torch.float64)
    for b, (n, kv) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        t = slice(s["start"][b], s["start"][b] + n)
        k, v = [ref.rows_of(s[x], s["table"], b, kv, s["page"]).float() for x in ("k", "v")]
        hidden = torch.arange(kv)[None, :] > torch.arange(kv - n, kv)[:, None]
        for h in range(s["heads"]):
            x = (s["q"][t, h].float() @ k[h // group].T) * s["dim"] ** -0.5
            x = x.masked_fill(hidden, float("-inf"))
            lift = 2.0 ** 7 if dtype is torch.float16 else 1.0
            p = torch.exp(x - x.amax(-1, keepdim=True)) * lift
            r = p.to(dtype).float()
            total = (r if sum_of_rounded else p).sum(-1, keepdim=True)
            out[t, h] = ((r @ v[h // group]) / total).to(dtype).double()
    return out


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("kind,q_lens,kv_lens", pb.PEAKED)
@pytest.mark.parametrize("q_factor,key_factor", [(1, 1), (8, 1), (40, 1), (40, 100)])
def test_bound(dt, kind, q_lens, kv_lens, q_factor, key_factor):
    s = pb.peaked_batch(q_lens, kv_lens, dt, q_factor, key_factor, device="cpu")
    for rounded in (True, False):
        want, bound = pb.attention(s, sum_of_rounded=rounded)
        assert bool(bound.isfinite().all())
        assert bool(((emulate(s, rounded) - want).abs() <= bound).all())
        # wrong outputs are noticed. All zeros: an even row's outputs are averages of some 150 normal values,
        # 0.08 wide, and the widest bound (bf16) is 0.007, so 7 % of them lie within it.
        assert float((want.abs() <= bound).double().mean()) < 0.1
        # one value row left out, where its key takes about half of the rows whole
        less = {**s, "v": s["v"].clone()}
        less["v"][int(s["table"][0, 0]), :, 3] = 0
        off = (emulate(less, rounded) - want).abs() > bound
        if key_factor == 100:
            assert float(off[:q_lens[0]].double().mean()) > 0.3
