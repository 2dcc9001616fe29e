"""Plain 64-bit forms of the paged-cache operators and the inputs of their tests."""
import math

import torch

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype):
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def make_batch(q_lens, kv_lens, heads=8, kv_heads=2, dim=128, page=16, dt="bf16", layout="hnd", seed=0, junk=True,
               q_std=1.5, spare_rows=0, device="cuda"):
    """A cache with shuffled pages and packed queries. junk: pages nobody owns
    and rows behind a sequence's end hold NaN, table entries behind its last
    page point nowhere. spare_rows: rows of q behind the last sequence."""
    g = torch.Generator(device=device).manual_seed(seed)
    dtype = DTYPES[dt]
    B = len(q_lens)
    need = [-(-kv // page) for kv in kv_lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=device).tolist()
    wide = max(need + [1]) + 2
    table = torch.full((B, wide), -7 if junk else 0, dtype=torch.int32)
    owned = []
    for b in range(B):
        for i in range(need[b]):
            table[b, i] = order[len(owned)]
            owned.append(order[len(owned)])

    def pool():
        shape = {"hnd": (pages, kv_heads, page, dim), "nhd": (pages, page, kv_heads, dim),
                 "padded": (pages, kv_heads, page, dim + 8)}[layout]
        x = torch.full(shape, float("nan"), device=device, dtype=dtype)
        x = {"hnd": lambda: x, "nhd": lambda: x.transpose(1, 2), "padded": lambda: x[..., :dim]}[layout]()
        fill = torch.randn((pages, kv_heads, page, dim), generator=g, device=device).to(dtype)
        if not junk:
            x.copy_(fill)
            return x
        for b in range(B):
            for i in range(need[b]):
                n = min(page, kv_lens[b] - i * page)
                at = int(table[b, i])
                x[at, :, :n] = fill[at, :, :n]
        return x

    start = [0]
    for n in q_lens:
        start.append(start[-1] + n)
    q = (q_std * torch.randn((start[-1] + spare_rows, heads, dim), generator=g, device=device)).to(dtype)
    return {"q": q, "k": pool(), "v": pool(), "table": table.to(device), "q_lens": list(q_lens),
            "kv_lens": list(kv_lens), "start": start, "page": page, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "q_start": torch.tensor(start, dtype=torch.int32, device=device),
            "kv_len": torch.tensor(kv_lens, dtype=torch.int32, device=device)}


def rows_of(pool, table, b, kv, page):
    """Sequence b's cached rows, [kv_heads, kv, dim]."""
    at = table[b, :-(-kv // page)].long()
    x = pool[at].transpose(0, 1)
    return x.reshape(x.shape[0], -1, x.shape[3])[:, :kv]


def attention(s, window=0, sinks=0, scale=None):
    """(out [T, heads, dim], bound) in 64 bits. The bound on a kernel's error,
    with u the half step of the storage type and A = sum p |v| / sum p:
      u (A + |o|)   p rounded before the product, the sum taking rounded p's
                    (or u A where it takes unrounded ones)
      u |o|         the output's rounding
      2 A e         e the relative error of a p in fp32: the score's dot product
                    (D + 2 terms of 2^-23 of sum |q_i k_i|), its scaling and the
                    exponential (2^-18), and the running sums of n terms (n / 16
                    steps and 64 joins of 2^-23, on both sums)."""
    dim, group = s["dim"], s["heads"] // s["kv_heads"]
    scale = dim ** -0.5 if scale is None else scale
    u = half_step(s["q"].dtype)
    out = torch.zeros((s["start"][-1], s["heads"], dim), dtype=torch.float64, device=s["q"].device)
    bound = torch.zeros_like(out)
    for b, (n, kv) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        if n == 0 or kv == 0:
            continue
        t = slice(s["start"][b], s["start"][b] + n)
        k = rows_of(s["k"], s["table"], b, kv, s["page"]).double().repeat_interleave(group, 0)
        v = rows_of(s["v"], s["table"], b, kv, s["page"]).double().repeat_interleave(group, 0)
        q = s["q"][t].double().transpose(0, 1)
        p = torch.arange(kv - n, kv, device=k.device)[:, None]
        j = torch.arange(kv, device=k.device)[None, :]
        seen = j <= p
        if window:
            seen &= (p - j < window) | (j < sinks)
        union = seen.any(0)
        k, v = k.clone(), v.clone()
        k[:, ~union], v[:, ~union] = 0, 0
        x = (q @ k.transpose(1, 2)) * scale
        x = x.masked_fill(~seen, float("-inf"))
        m = x.amax(-1, keepdim=True)
        e = torch.exp(x - torch.where(m == float("-inf"), torch.zeros_like(m), m))
        total = e.sum(-1, keepdim=True).clamp(min=1e-300)
        o = (e @ v) / total
        A = (e @ v.abs()) / total
        dots = (q.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * abs(scale)
        err = (dim + 2) * 2.0 ** -23 * dots + 2.0 ** -18 + (kv / 16 + 64) * 2.0 ** -23
        out[t] = o.transpose(0, 1)
        bound[t] = (u * (A + 2 * o.abs()) + 2 * A * err).transpose(0, 1)
    tiny = torch.finfo(s["q"].dtype).smallest_normal * torch.finfo(s["q"].dtype).eps
    return out, bound + tiny


def norm_rope(x, weight, cos, sin, pos, eps):
    """Per-head norm and rotation of x [n, heads, dim] at positions pos, 64 bits."""
    x = x.double()
    dim = x.shape[-1]
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    if cos is None:
        return x
    c, z = cos[pos].double()[:, None], sin[pos].double()[:, None]
    a, b = x[..., :dim // 2], x[..., dim // 2:]
    return torch.cat([a * c - b * z, b * c + a * z], -1)


def sample_row(x, t, k, p, low, u):
    """(id, logprob, margin) of one row of logits (python floats and ints):
    margin is how far, relative to the kept mass, u or a cut is from the
    nearest border."""
    n = len(x)
    order = sorted((i for i in range(n) if not math.isnan(x[i]) and x[i] != -math.inf), key=lambda i: (-x[i], i))
    if not order:
        return -1, -math.inf, 1.0
    if not t > 0:
        return order[0], 0.0, 1.0
    top = x[order[0]]
    w = [1.0 if x[i] == top else (0.0 if top == math.inf else math.exp((x[i] - top) / t)) for i in order]
    if 0 < k < len(w):
        w = w[:k]
    margin = 1.0
    if not p >= 1:
        goal, run, kept = p * math.fsum(w), 0.0, 0
        while kept < len(w) and (kept == 0 or run < goal):
            run += w[kept]
            kept += 1
            margin = min(margin, abs(run - goal) / goal if goal > 0 else 1.0)
        w = w[:kept]
    w = [w[0]] + [y for y in w[1:] if y >= low]
    total = math.fsum(w)
    run = 0.0
    for i, y in enumerate(w):
        run += y
        margin = min(margin, abs(run - u * total) / total)
        if run > u * total:
            break
    return order[i], math.log(w[i] / total) if w[i] > 0 else -math.inf, margin
