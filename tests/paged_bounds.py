"""Error bound of the paged attention kernels that follows each key's own error.

With w_j a key's weight, x_j its scaled score, and p_j the kernel's e^(x_j - m)
off by a factor 1 + d_j, an output whose sum takes the same p_j is off by

  sum_j w_j d_j (v_j - o) / (1 + sum_j w_j d_j)

to all orders: a factor that all keys share cancels, so a row that one key
takes whole is exact however far off that key's score is. |d_j| is bounded from

  (D + 2) 2^-23 S_j           the dot product in fp32, S_j = |scale| sum_i |q_i k_ij|
  2^-22 (max |x| + |x_j|)     scale * log2 e rounded, the product, the maximum's
                              and the difference's rounding, 2^-24 each
  2^-21                       the exponential: ex2.approx 2^-22, the polynomial 2^-22.1
  u                           p rounded to the storage type (u its half step)

and the output adds

  u |o|                       its own rounding
  2 A (kv / 16 + 64) 2^-23    the running sums of both, 16 keys a step, and their joins
  2^-32 sum_j |v_j - o|       fp16: half a subnormal step of p, whose largest is at least 2^7
  u A                         only where the sum takes p before its rounding
"""
import torch

import paged_ref as ref


def _spread(w, d, gap):
    """sum w d |v - o| / (1 - sum w d), infinite where the denominator is below a half."""
    off = (w * d).sum(-1, keepdim=True)
    s = ((w * d)[:, :, None] * gap).sum(1)
    return torch.where(off < 0.5, s / (1 - off.clamp(max=0.5)), torch.full_like(s, float("inf")))


def attention(s, window=0, sinks=0, scale=None, sum_of_rounded=True):
    """(out [T, heads, dim], bound) in 64 bits; small batches (rows x keys x dim values a head)."""
    dim, group, page = s["dim"], s["heads"] // s["kv_heads"], s["page"]
    scale = dim ** -0.5 if scale is None else scale
    dtype, dev = s["q"].dtype, s["q"].device
    u = ref.half_step(dtype)
    out = torch.zeros((s["start"][-1], s["heads"], dim), dtype=torch.float64, device=dev)
    bound = torch.zeros_like(out)
    for b, (n, kv) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        if n == 0 or kv == 0:
            continue
        t = slice(s["start"][b], s["start"][b] + n)
        pos = torch.arange(kv - n, kv, device=dev)[:, None]
        j = torch.arange(kv, device=dev)[None, :]
        seen = j <= pos
        if window:
            seen &= (pos - j < window) | (j < sinks)
        keys, values = [ref.rows_of(s[x], s["table"], b, kv, page).double() for x in ("k", "v")]
        for h in range(s["heads"]):
            q, k, v = s["q"][t, h].double(), keys[h // group], values[h // group]
            x = (q @ k.T * scale).masked_fill(~seen, float("-inf"))
            top, r = x.max(-1, keepdim=True)
            w = torch.exp(x - top)
            w = w / w.sum(-1, keepdim=True)
            o = w @ v
            A = w @ v.abs()
            size = x.abs().masked_fill(~seen, 0.0)
            e = (dim + 2) * 2.0 ** -23 * abs(scale) * (q.abs() @ k.abs().T) + \
                2.0 ** -22 * (size.amax(-1, keepdim=True) + size) + 2.0 ** -21
            gap = (v[None] - o[:, None]).abs() * seen[:, :, None]
            alone = torch.expm1(e) * (1 + u) + u
            # errors relative to the first of the largest weights
            beside = (torch.expm1(e + e.gather(1, r)) * (1 + 2 * u) + 2.1 * u).scatter(1, r, 0.0)
            y = torch.minimum(_spread(w, alone, gap), _spread(w, beside, gap))
            y = y + u * o.abs() * (1 + u) + 2 * A * (kv / 16 + 64) * 2.0 ** -23
            if not sum_of_rounded:
                y = y + u * A
            if dtype is torch.float16:
                y = y + 2.0 ** -32 * gap.sum(1)
            out[t, h], bound[t, h] = o, y
    return out, bound + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


# Inputs whose rows are far from even: scores of a wide spread, and one key that
# takes the rows it points along and vanishes from the others.
PEAKED = [("few", [1, 1], [900, 80]), ("few", [5], [261]), ("few", [2, 3], [33, 600]),
          ("chunk", [90, 2], [300, 40]), ("chunk", [64], [500]), ("chunk", [33], [65])]


def peaked_batch(q_lens, kv_lens, dt, q_factor, key_factor, dim=128, device="cuda"):
    s = ref.make_batch(q_lens, kv_lens, heads=4, kv_heads=1, dim=dim, dt=dt, seed=8, device=device)
    s["q"].mul_(q_factor)
    s["k"][int(s["table"][0, 0]), :, 3] *= key_factor
    return s
