"""The operators of serving from a paged key/value cache: their inputs, plain forms and calls.

Three operators, as one step of a serving loop uses them:

  norm_rope  the new tokens' queries and keys are normalised for each head and rotated, and the keys and values go to
             their rows of the cache's pages;
  attention  each new token attends its sequence's cached rows through the page table (one token or a chunk of them
             for each sequence, grouped query heads, optionally a sliding window with a few first rows kept visible);
  sample     one token id for each row of logits, from temperature, top-k, top-p and min-p and a given random number.

Shapes. A cache layer is two tensors [pages, kv_heads, page_size, head_dim]; sequence b's row j is row j % page_size of
page page_table[b, j // page_size]. The call's tokens are packed: sequence b has rows q_start[b] .. q_start[b + 1] - 1,
and they sit at the last positions of its kv_len[b] rows.

`run` computes them with elementary torch operations, or with the framework's entry points where `own` is true.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
ROPE_THETA = 500000.0


# ------------------------------------------------------------------ cases
def _attention(name, dtype, batch, q, kv, lens, heads=32, kv_heads=8, head_dim=128, page=16, window=0, sinks=0):
    """lens: "same" (every sequence q new tokens, kv rows), "ragged" (up to q, up to kv) or "mixed" (one sequence in
    three brings a chunk of up to q tokens, the others one token each)."""
    return {"name": name, "op": "attention", "dtype": dtype, "batch": batch, "q": q, "kv": kv, "lens": lens,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "window": window,
            "sinks": sinks}


def _norm_rope(name, dtype, batch, q, kv, lens, heads=32, kv_heads=8, head_dim=128, page=16):
    return {"name": name, "op": "norm_rope", "dtype": dtype, "batch": batch, "q": q, "kv": kv, "lens": lens,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page}


def _sample(name, dtype, batch, vocab):
    return {"name": name, "op": "sample", "dtype": dtype, "batch": batch, "vocab": vocab}


def listed():
    return [
        # one user's decode step after the 2048-token prompt of the benchmark: latency
        _attention("decode_one", "bf16", 1, 1, 2049, "same"),
        # a full decode batch of a server, every context length from a few tokens to 8192
        _attention("decode_ragged", "bf16", 64, 1, 8192, "ragged"),
        # one token over a very long context: the rows have to be split over the whole GPU
        _attention("decode_long", "f16", 1, 1, 131071, "same", page=64),
        # speculative verification: 4 draft tokens + 1 for each of eight sequences
        _attention("verify", "bf16", 8, 5, 2053, "ragged"),
        # a whole 2048-token prompt in one call
        _attention("prefill", "bf16", 1, 2048, 2048, "same"),
        # chunked prefill next to decoding sequences, ragged
        _attention("mixed", "f16", 12, 1024, 8191, "mixed", page=32),
        # a long chunk of a sliding-window layer with four sink rows, heads of 64
        _attention("window", "bf16", 2, 4096, 12345, "same", heads=16, kv_heads=2, head_dim=64, page=64,
                   window=1024, sinks=4),
        # one decode step of eight sequences: latency
        _norm_rope("norm_rope_decode", "bf16", 8, 1, 2048, "ragged"),
        # the tokens of a large prefill batch: bandwidth
        _norm_rope("norm_rope_prefill", "f16", 5, 4095, 4095, "ragged", page=32),
        # the next token of one user
        _sample("sample_one", "bf16", 1, 128256),
        # the next tokens of a decode batch
        _sample("sample_batch", "bf16", 64, 128256),
        # a large batch over a smaller vocabulary of odd size
        _sample("sample_wide", "f16", 250, 50257),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "norm_rope", "sample"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "sample":
        case = _sample("", dtype, _log_int(rng, 1, 250), _log_int(rng, 1000, 128256))
        while case["batch"] * case["vocab"] > 250 * 50257:
            case["batch"] //= 2
    else:
        kv_heads = rng.choice([1, 2, 4, 8])
        shape = {"heads": kv_heads * rng.choice([1, 2, 3, 4, 8]), "kv_heads": kv_heads,
                 "head_dim": rng.choice([64, 128]), "page": rng.choice([16, 32, 64, 128])}
        if op == "norm_rope":
            q = _log_int(rng, 1, 4095)
            case = _norm_rope("", dtype, _log_int(rng, 1, 64), q, q + _log_int(rng, 1, 4096),
                              rng.choice(["same", "ragged", "mixed"]), **shape)
            while case["batch"] * case["q"] * (case["heads"] + 2 * case["kv_heads"]) > 5 * 4095 * 40:
                case["batch"] = max(1, case["batch"] // 2)
                case["q"] = max(1, case["q"] // 2)
        else:
            q = rng.choice([1, rng.randint(2, 8), _log_int(rng, 9, 4096)])
            kv = q + _log_int(rng, 1, 131071 if q == 1 else 8191)
            window, sinks = rng.choice([(0, 0), (0, 0), (_log_int(rng, 16, 4096), rng.choice([0, 4, 17]))])
            case = _attention("", dtype, _log_int(rng, 1, 64), q, kv, rng.choice(["same", "ragged", "mixed"]),
                              window=window, sinks=sinks, **shape)
            while (case["batch"] * case["kv"] * case["kv_heads"] > 64 * 8192 * 8
                   or case["batch"] * case["q"] * case["kv"] * case["heads"] > 12 * 1024 * 8192 * 32):
                if case["batch"] > 1:
                    case["batch"] //= 2
                else:
                    case["q"] = max(1, case["q"] // 2)
                    case["kv"] = max(case["q"], case["kv"] // 2)
    del case["name"]
    return case


def _lengths(case):
    """(new tokens, cached rows with them) of each sequence: a function of the case alone."""
    rng = random.Random("%s %s %s %s" % (case["batch"], case["q"], case["kv"], case["lens"]))
    pairs = []
    for b in range(case["batch"]):
        q, kv = case["q"], case["kv"]
        if b and case["lens"] == "mixed":
            q = _log_int(rng, 1, q) if b % 3 == 0 else 1
            kv = max(q, _log_int(rng, 1, kv))
        elif b and case["lens"] == "ragged":
            kv = max(1, rng.randint(1, kv))
            q = min(q, kv) if q <= 8 else min(kv, rng.randint(1, q))
        pairs.append((q, kv))
    return pairs


def _seen(q, kv, window, sinks):
    """(rows of the cache that some new token sees, visible (token, row) pairs) of one sequence."""
    if not window:
        return kv, q * (kv - q) + q * (q + 1) // 2
    first = max(0, kv - q - window + 1)
    rows = kv - first + min(sinks, first)
    pairs = 0
    for p in range(kv - q, kv):
        start = max(0, p - window + 1)
        pairs += p + 1 - start + min(sinks, start)
    return rows, pairs


def work(case):
    if case["op"] == "sample":
        n = case["batch"] * case["vocab"]
        # each logit is read once, compared, exponentiated and added; 20 bytes of parameters and 8 of results a row
        return {"bytes": 2 * n + 28 * case["batch"], "flops": 4 * n}
    lens = _lengths(case)
    tokens = sum(q for q, _ in lens)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    table = 4 * (2 * len(lens) + 1 + sum(-(-kv // case["page"]) for _, kv in lens))
    if case["op"] == "norm_rope":
        # q, k and v read once and written once, a row of the two rotation tables for each position
        return {"bytes": 4 * tokens * (heads + 2 * kv_heads) * dim + 4 * tokens * dim + table,
                "flops": tokens * (heads + kv_heads) * dim * 8}
    seen = [_seen(q, kv, case["window"], case["sinks"]) for q, kv in lens]
    rows, pairs = sum(r for r, _ in seen), sum(p for _, p in seen)
    return {"bytes": 4 * rows * kv_heads * dim + 4 * tokens * heads * dim + table, "flops": 4 * pairs * heads * dim}


# ----------------------------------------------------------------- inputs
def _normal(g, shape, dtype, std=1.0):
    x = torch.empty(shape, dtype=dtype, device="cuda")
    return x.normal_(0.0, std, generator=g)


def _sequences(case, g):
    """The cache, its page table and the sequences' extents: pages in random order, with some that nobody owns."""
    lens, page = _lengths(case), case["page"]
    need = [-(-kv // page) for _, kv in lens]
    owned = sum(need)
    pages = owned + owned // 8 + 1
    order = torch.randperm(pages, generator=g, device="cuda")[:owned].to(torch.int32)
    wide = max(need)
    slot = torch.arange(wide, device="cuda")[None, :]
    counts = torch.tensor(need, device="cuda")[:, None]
    first = torch.cumsum(counts, 0) - counts
    table = torch.where(slot < counts, order[(first + slot).clamp(max=owned - 1)], torch.zeros_like(order[:1]))
    starts = [0]
    for q, _ in lens:
        starts.append(starts[-1] + q)
    return {"pages": pages, "table": table.contiguous(), "tokens": starts[-1], "max_q": max(q for q, _ in lens),
            "max_kv": max(kv for _, kv in lens),
            "q_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
            "kv_len": torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "sample":
        rows, vocab = case["batch"], case["vocab"]
        # a language model's logits: a broad bulk and a few dozen likely tokens well above it
        logits = torch.empty(rows, vocab, device="cuda").normal_(0.0, 2.0, generator=g)
        likely = torch.randint(0, vocab, (rows, 40), generator=g, device="cuda")
        lift = torch.empty(rows, 40, device="cuda").exponential_(0.4, generator=g) + 6.0
        s["logits"] = logits.scatter(1, likely, lift).to(dtype)
        pick = lambda values, kind: torch.tensor(values, dtype=kind, device="cuda")[  # noqa: E731
            torch.randint(0, len(values), (rows,), generator=g, device="cuda")]
        s["temperature"] = pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3], torch.float32)
        s["top_k"] = pick([0, 0, 20, 50, 1000], torch.int32)
        s["top_p"] = pick([1.0, 0.8, 0.9, 0.95], torch.float32)
        s["min_p"] = pick([0.0, 0.0, 0.02, 0.1], torch.float32)
        s["u"] = torch.rand(rows, generator=g, device="cuda")
        if own:
            s["idx"] = torch.empty(rows, dtype=torch.int32, device="cuda")
            s["logprob"] = torch.empty(rows, dtype=torch.float32, device="cuda")
        return s
    s |= _sequences(case, g)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    layer = (s["pages"], kv_heads, case["page"], dim)
    s["k"], s["v"] = _normal(g, layer, dtype), _normal(g, layer, dtype)
    if case["op"] == "attention":
        s["q"] = _normal(g, (s["tokens"], heads, dim), dtype, 2.0)
        if own:
            import infengine_b200 as ie
            s["cache"] = ie.PagedCache(s["k"], s["v"])
            s["out"] = torch.empty(s["tokens"], heads * dim, dtype=dtype, device="cuda")
            s["workspace"] = ie.paged_attention_workspace()
        return s
    # q, k and v as columns of one projection's output
    fused = _normal(g, (s["tokens"], heads + 2 * kv_heads, dim), dtype, 1.5)
    s["q"], s["new_k"], s["new_v"] = fused[:, :heads], fused[:, heads:heads + kv_heads], fused[:, heads + kv_heads:]
    s["q_weight"] = (1.0 + 0.2 * _normal(g, (dim,), torch.float32)).to(dtype)
    s["k_weight"] = (1.0 + 0.2 * _normal(g, (dim,), torch.float32)).to(dtype)
    inv = ROPE_THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    angle = torch.arange(s["max_kv"], dtype=torch.float64, device="cuda")[:, None] * inv
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    if own:
        import infengine_b200 as ie
        s["cache"] = ie.PagedCache(s["k"], s["v"])
        s["q_out"] = torch.empty(s["tokens"], heads, dim, dtype=dtype, device="cuda")
    return s


# ------------------------------------------------------------ plain forms
def _owners(s):
    """For each new token: its sequence, its index there and its position."""
    token = torch.arange(s["tokens"], device="cuda")
    start = s["q_start"].long()
    seq = torch.searchsorted(start[1:], token, right=True)
    local = token - start[seq]
    return seq, local, s["kv_len"].long()[seq] - (start[seq + 1] - start[seq]) + local


def _plain_attention(s):
    case = s["case"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    group, batch, max_q = heads // kv_heads, case["batch"], s["max_q"]
    blocks = -(-s["max_kv"] // page)
    rows = blocks * page
    table = s["table"][:, :blocks].long()
    kv_len, start = s["kv_len"].long(), s["q_start"].long()
    key = torch.arange(rows, device="cuda")
    k = s["k"][table].float().transpose(2, 3).reshape(batch, rows, kv_heads, dim)
    v = s["v"][table].float().transpose(2, 3).reshape(batch, rows, kv_heads, dim)
    v = torch.where((key < kv_len[:, None])[:, :, None, None], v, torch.zeros((), device="cuda"))
    local = torch.arange(max_q, device="cuda")
    q = s["q"].float()[(start[:-1, None] + local).clamp(max=s["tokens"] - 1)]
    q = q.reshape(batch, max_q, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * max_q, dim)
    pos = (kv_len - (start[1:] - start[:-1]))[:, None] + local
    gap = pos[:, :, None] - key
    seen = (gap >= 0) & (key < kv_len[:, None])[:, None, :]
    if case["window"]:
        seen &= (gap < case["window"]) | (key < case["sinks"])
    score = torch.matmul(q, k.permute(0, 2, 3, 1)).reshape(batch, kv_heads, group, max_q, rows)
    score.mul_(1.0 / math.sqrt(dim)).masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.reshape(batch, kv_heads, group * max_q, rows), v.transpose(1, 2))
    o = o.reshape(batch, kv_heads, group, max_q, dim) / total.clamp(min=torch.finfo(torch.float32).tiny)
    seq, at, _ = _owners(s)
    return o.permute(0, 3, 1, 2, 4)[seq, at].reshape(s["tokens"], heads * dim).to(DTYPES[case["dtype"]])


def _plain_norm_rope(s):
    dtype, page = s["q"].dtype, s["case"]["page"]
    seq, _, pos = _owners(s)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turned(x, weight):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(dtype)

    at, row = s["table"].long()[seq, pos // page], pos % page
    s["k"][at, :, row] = turned(s["new_k"], s["k_weight"])
    s["v"][at, :, row] = s["new_v"]
    return {"q": turned(s["q"], s["q_weight"]), "k": s["k"], "v": s["v"]}


def _plain_sample(s):
    # 64 bits: the result turns on which side of a border a cumulative sum falls
    value, index = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)
    column = lambda x: x.double()[:, None]  # noqa: E731
    t, vocab = column(s["temperature"]), value.shape[1]
    greedy = ~(t > 0)
    ratio = torch.exp((value - value[:, :1]) / torch.where(greedy, torch.ones_like(t), t))
    rank = torch.arange(vocab, device="cuda")
    k = s["top_k"].long()[:, None]
    k = torch.where((k <= 0) | (k > vocab), torch.full_like(k, vocab), k)
    weight = torch.where((rank < k) & (~greedy | (rank < 1)), ratio, torch.zeros_like(ratio))
    total = weight.cumsum(-1)
    before = total - weight
    p, low = column(s["top_p"]), column(s["min_p"])
    kept = (rank < 1) | (((before < p * total[:, -1:]) | (p >= 1)) & (ratio >= low))
    weight = torch.where(kept, weight, torch.zeros_like(weight))
    total = weight.cumsum(-1)
    target = column(s["u"]) * total[:, -1:]
    last = (weight > 0).sum(-1, keepdim=True) - 1
    at = torch.minimum((total <= target).sum(-1, keepdim=True), last)
    logprob = torch.log(weight.gather(1, at) / total[:, -1:])
    return {"idx": index.gather(1, at)[:, 0].int(), "logprob": logprob[:, 0].float()}


def run(s):
    case = s["case"]
    if not own:
        return {"attention": _plain_attention, "norm_rope": _plain_norm_rope, "sample": _plain_sample}[case["op"]](s)
    import infengine_b200 as ie
    if case["op"] == "attention":
        ie.paged_attention(s["q"], s["cache"], s["table"], s["q_start"], s["kv_len"], s["out"], max_q=s["max_q"],
                           window=case["window"], sinks=case["sinks"], workspace=s["workspace"])
        return s["out"]
    if case["op"] == "norm_rope":
        ie.qk_norm_rope_paged(s["q"], s["new_k"], s["new_v"], s["q_weight"], s["k_weight"], s["cos"], s["sin"],
                              s["cache"], s["table"], s["q_start"], s["kv_len"], s["q_out"], eps=EPS)
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    ie.sample(s["logits"], s["u"], s["idx"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
              min_p=s["min_p"], logprob_out=s["logprob"])
    return {"idx": s["idx"], "logprob": s["logprob"]}


# ------------------------------------------------------- definitions, 64 bits
def _exact_attention(s):
    case = s["case"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros(s["tokens"], heads, dim, dtype=torch.float64, device="cuda")
    begin = 0
    for b, (n, kv) in enumerate(_lengths(case)):
        pages = s["table"][b, :-(-kv // page)].long()
        p = torch.arange(kv - n, kv, device="cuda")[:, None]
        j = torch.arange(kv, device="cuda")[None, :]
        hidden = j > p
        if case["window"]:
            hidden |= (p - j >= case["window"]) & (j >= case["sinks"])
        for h in range(kv_heads):
            keys = s["k"][pages, h].reshape(-1, dim)[:kv].double()
            values = s["v"][pages, h].reshape(-1, dim)[:kv].double()
            for head in range(h * (heads // kv_heads), (h + 1) * (heads // kv_heads)):
                x = s["q"][begin:begin + n, head].double() @ keys.T / math.sqrt(dim)
                x = x.masked_fill(hidden, float("-inf"))
                e = torch.exp(x - x.max(1, keepdim=True).values)
                out[begin:begin + n, head] = (e @ values) / e.sum(1, keepdim=True)
        begin += n
    return out.reshape(s["tokens"], heads * dim)


def _exact_norm_rope(s):
    dim, page = s["case"]["head_dim"], s["case"]["page"]
    k, v, q = s["k"].double(), s["v"].double(), torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    half = dim // 2

    def rows(x, w, p):
        x = x.double()
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / dim + EPS) * w.double()
        c, z = s["cos"][p].double()[:, None, :], s["sin"][p].double()[:, None, :]
        y = torch.empty_like(x)
        y[..., :half] = x[..., :half] * c - x[..., half:] * z
        y[..., half:] = x[..., half:] * c + x[..., :half] * z
        return y

    begin = 0
    for b, (n, kv) in enumerate(_lengths(s["case"])):
        p = torch.arange(kv - n, kv, device="cuda")
        t = slice(begin, begin + n)
        q[t] = rows(s["q"][t], s["q_weight"], p)
        at = s["table"][b].long()[p // page]
        k[at, :, p % page] = rows(s["new_k"][t], s["k_weight"], p)
        v[at, :, p % page] = s["new_v"][t].double()
        begin += n
    return {"q": q, "k": k, "v": v}


def _exact_sample(s):
    rows = []
    for r in range(s["logits"].shape[0]):
        x = s["logits"][r].double()
        t, k = float(s["temperature"][r]), int(s["top_k"][r])
        p, low, u = float(s["top_p"][r]), float(s["min_p"][r]), float(s["u"][r])
        if not t > 0:
            rows.append((int((x == x.max()).nonzero()[0, 0]), 0.0))
            continue
        order = torch.argsort(-x, stable=True)
        w = torch.exp((x[order] - x.max()) / t)
        relative = w
        if 0 < k < len(w):
            w = w[:k]
        sums = torch.cumsum(w, 0)
        n = len(w)
        if p < 1:
            n = 1 + int((sums[:-1] < p * sums[-1]).sum())
        n = max(1, min(n, int((relative[:n] >= low).sum())))
        sums = sums[:n]
        i = min(int((sums <= u * sums[-1]).sum()), n - 1)
        rows.append((int(order[i]), float(torch.log(w[i] / sums[-1]))))
    return {"idx": torch.tensor([i for i, _ in rows], dtype=torch.int32, device="cuda"),
            "logprob": torch.tensor([x for _, x in rows], dtype=torch.float64, device="cuda")}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "norm_rope": _exact_norm_rope, "sample": _exact_sample}[case["op"]](s)
