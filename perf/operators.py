"""Cases that measure the operators of a decode step on 4-bit caches.

A server that keeps its sequences' keys and values in 4 bits runs, per layer and step,

* ``norms``:   the norms of queries and keys for each head, with the position rotation in the same pass;
* ``append``:  the same with the keys and values stored in the 4-bit cache instead of returned (the rows are read
  back here, since what a cache holds is its output);
* ``attend``:  attention over the 4-bit cache, one query per sequence or a chunk of a prompt, with an optional sliding
  window whose first tokens (sinks) stay visible;

and, after the head matrix,

* ``sample``:  a token per sequence by temperature, top-k, top-p and min-p from given random numbers.

``run`` computes them in plain torch (``own`` false) or with blocktensor_b200 (``own`` true).

The cache: a page holds ``[kv_heads][page][row]`` rows, one array for K and one for V.  A row is head_dim / 2 bytes
of codes (element 2i in the low nibble of byte i), then a (scale, min) pair of fp16 for every 64 elements; a code c
stands for scale * c + min.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GROUP = 64            # elements that share a (scale, min) pair
LIMIT = 57344.0       # values are held to +-LIMIT, so that scale * 15 + min stays inside fp16
UNIT = float(2 ** 40)  # sampling weights are whole multiples of 2^-40 of the largest one


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one token of the 7B shape (multi-head), fp32 activations as the engine's: all launch latency
        dict(name="norms 7B token", op="norms", tokens=1, heads=32, kv_heads=32, head_dim=128, dtype="f32", rot=128),
        # a prompt of the 70B shape out of a fused q/k/v product: all bandwidth
        dict(name="norms 70B prompt", op="norms", tokens=8192, heads=64, kv_heads=8, head_dim=128, dtype="bf16", rot=128),
        # one step of 64 TinyLlama-shaped sequences into 64-position pages
        dict(name="append TinyLlama batch", op="append", tokens=64, heads=32, kv_heads=4, head_dim=64, dtype="f32",
             rot=64, page=64, spread=True),
        # a prompt of the 70B shape into its cache
        dict(name="append 70B prompt", op="append", tokens=4099, heads=64, kv_heads=8, head_dim=128, dtype="bf16",
             rot=128, page=0, spread=False),
        # single-sequence decode of the 7B shape behind a 512-token prompt, fp32 queries
        dict(name="attend 7B token", op="attend", n=1, q_lo=1, q_hi=1, len_lo=550, len_hi=550, heads=32, kv_heads=32,
             head_dim=128, dtype="f32", page=0, window=0, sinks=0),
        # batched decode: 64 TinyLlama-shaped sequences, contexts 128 to 4096, paged
        dict(name="attend TinyLlama batch", op="attend", n=64, q_lo=1, q_hi=1, len_lo=128, len_hi=4096, heads=32,
             kv_heads=4, head_dim=64, dtype="f16", page=64, window=0, sinks=0),
        # decode of long sequences through a window of 4096 with 4 sinks, 70B shape
        dict(name="attend 70B window", op="attend", n=24, q_lo=1, q_hi=1, len_lo=5000, len_hi=65531, heads=64,
             kv_heads=8, head_dim=128, dtype="bf16", page=256, window=4096, sinks=4),
        # one very long sequence alone on the GPU
        dict(name="attend 70B long token", op="attend", n=1, q_lo=1, q_hi=1, len_lo=131071, len_hi=131071, heads=64,
             kv_heads=8, head_dim=128, dtype="bf16", page=0, window=0, sinks=0),
        # prompts of uneven lengths prefilled together, TinyLlama shape
        dict(name="attend TinyLlama prompts", op="attend", n=8, q_lo=1, q_hi=1531, len_lo=1, len_hi=1531, heads=32,
             kv_heads=4, head_dim=64, dtype="f16", page=64, window=512, sinks=4),
        # a 2048-token chunk of an 8192-token prompt, 70B shape
        dict(name="attend 70B chunk", op="attend", n=1, q_lo=2048, q_hi=2048, len_lo=8192, len_hi=8192, heads=64,
             kv_heads=8, head_dim=128, dtype="bf16", page=0, window=0, sinks=0),
        # one sequence's next token
        dict(name="sample one", op="sample", rows=1, vocab=32000, dtype="f32", top_k=40, filters="all"),
        # a batch with requests of all kinds over the 70B shape's vocabulary
        dict(name="sample batch", op="sample", rows=256, vocab=128256, dtype="f32", top_k=50, filters="mixed"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norms", "append", "attend", "attend", "sample"])
    head_dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
    group = rng.choice([1, 2, 4, 5, 8, 12])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op in ("norms", "append"):
        most = max(2, 8192 * 72 * 128 // ((kv_heads * group + 2 * kv_heads) * head_dim * (2 if op == "append" else 1)))
        case = dict(op=op, tokens=_log_int(rng, 1, min(16384, most)), heads=kv_heads * group, kv_heads=kv_heads,
                    head_dim=head_dim, dtype=dtype, rot=rng.choice([head_dim, head_dim, head_dim // 2]))
        if op == "append":
            case.update(page=rng.choice([0, 16, 64, 256]), spread=rng.random() < 0.5)
        return case
    if op == "attend":
        window = rng.choice([0, 0, _log_int(rng, 1, 4096)])
        sinks = rng.choice([0, 1, 4, 37]) if window else 0
        page = rng.choice([0, 16, 64, 128, 1024])
        if rng.random() < 0.5:  # single tokens
            n = _log_int(rng, 1, 128)
            most = max(64, min(131072, (1 << 27) // (n * kv_heads * head_dim)))
            hi = _log_int(rng, 1, most)
            q_lo = q_hi = 1
        else:
            n = _log_int(rng, 1, 12)
            hi = _log_int(rng, 2, 8192)
            area = 1.0e9 if dtype != "f32" else 2.5e8  # scores of the plain form
            q_hi = _log_int(rng, 2, max(2, min(2048, hi, int(area / (n * kv_heads * group * hi)))))
            q_lo = rng.choice([1, q_hi])
        return dict(op=op, n=n, q_lo=q_lo, q_hi=q_hi, len_lo=rng.choice([min(1, hi), max(1, hi // 3), hi]), len_hi=hi,
                    heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, page=page,
                    window=window, sinks=sinks)
    vocab = _log_int(rng, 100, 262144)
    return dict(op=op, rows=_log_int(rng, 1, min(512, (1 << 25) // vocab)), vocab=vocab, dtype=dtype,
                top_k=_log_int(rng, 1, vocab), filters=rng.choice(["all", "mixed", "mixed", "none"]))


# ---------------------------------------------------------------- inputs

def _spaced(lo, hi, n):
    """n whole numbers from lo to hi, evenly spread and out of order."""
    at = [hi] if n == 1 else [lo + round(i * (hi - lo) / (n - 1)) for i in range(n)]
    return at[::2] + at[1::2][::-1]


def _lengths(case):
    """(queries, cached positions) of every sequence; the queries are the last positions."""
    lens = _spaced(case["len_lo"], case["len_hi"], case["n"])
    return [min(q, length) for q, length in zip(_spaced(case["q_lo"], case["q_hi"], case["n"]), lens)], lens


def _row_bytes(head_dim):
    return head_dim // 2 + head_dim // GROUP * 4


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _table(positions, rot, theta=500000.0):
    """cos and sin of every position and pair, [positions][rot / 2][2]."""
    inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def _cache(state, n, max_seq, kv_heads, head_dim, page, k_rows, v_rows, table):
    state.update(k_rows=k_rows, v_rows=v_rows, table=table)
    if own:
        import blocktensor_b200 as bt
        state["cache"] = bt.KV4Cache(n, max_seq, kv_heads, head_dim, page_tokens=page, k_rows=k_rows, v_rows=v_rows,
                                     page_table=table if page else None)


def _pages(case, g, n, max_seq):
    """Tokens of a page, pages in all, and the table [n][pages of a sequence] (a contiguous cache: one page each)."""
    size = case["page"] or -(-max_seq // 16) * 16
    each = -(-max_seq // size)
    order = torch.randperm(n * each, generator=g, device="cuda") if case["page"] else torch.arange(n * each, device="cuda")
    return size, n * each, order.view(n, each).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    state = dict(case)
    if case["op"] == "sample":
        return _prepare_sample(case, g, state)
    if case["op"] == "attend":
        return _prepare_attend(case, g, state)
    tokens, heads, kv_heads, head_dim = (case[k] for k in ("tokens", "heads", "kv_heads", "head_dim"))
    # the rows of a fused q/k/v product, some channels larger than others, as trained projections give them
    qkv = _normal(g, tokens, heads + 2 * kv_heads, head_dim) * (1 + 2 * torch.rand(head_dim, generator=g, device="cuda"))
    qkv = qkv.to(DTYPES[case["dtype"]])
    state["q"], state["k"], state["v"] = qkv.split([heads, kv_heads, kv_heads], 1)
    state["qw"], state["kw"] = (1 + 0.3 * _normal(g, 2, head_dim)).unbind(0)
    state["eps"] = 1e-5
    if case["op"] == "norms":
        state["positions"] = torch.arange(tokens, dtype=torch.int32, device="cuda") + (511 if tokens == 1 else 0)
        state["rope"] = _table(tokens + 511, case["rot"])
        return state
    n = tokens if case["spread"] else 1  # each token its own sequence (a step), or all of one (a prompt)
    max_seq = 4096 if case["spread"] else tokens + 7
    size, pages, table = _pages(case, g, n, max_seq if not case["spread"] else min(4096, max(64, 262144 // n)))
    max_seq = table.shape[1] * size
    if case["spread"]:
        state["slots"] = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
        state["positions"] = torch.randint(0, max_seq, (n,), generator=g, device="cuda", dtype=torch.int32)
    else:
        state["slots"] = torch.zeros(tokens, dtype=torch.int32, device="cuda")
        state["positions"] = torch.arange(7, tokens + 7, dtype=torch.int32, device="cuda")
    state["rope"] = _table(max_seq, case["rot"])
    k_rows, v_rows = torch.zeros(2, pages, kv_heads, size, _row_bytes(head_dim), dtype=torch.uint8, device="cuda").unbind(0)
    _cache(state, n, max_seq, kv_heads, head_dim, case["page"], k_rows, v_rows, table)
    return state


def _random_rows(g, pages, kv_heads, size, head_dim):
    """Cache rows as quantised activations leave them: codes over the whole range, scales around 0.3."""
    rows = torch.randint(0, 256, (pages, kv_heads, size, _row_bytes(head_dim)), generator=g, device="cuda", dtype=torch.uint8)
    groups = head_dim // GROUP
    scale = 0.2 + 0.2 * torch.rand(pages, kv_heads, size, groups, generator=g, device="cuda")
    low = -scale * (7.5 + 0.5 * torch.randn(pages, kv_heads, size, groups, generator=g, device="cuda"))
    rows[..., head_dim // 2:] = torch.stack([scale, low], -1).half().flatten(-2).view(torch.uint8)
    return rows


def _prepare_attend(case, g, state):
    n, heads, kv_heads, head_dim = (case[k] for k in ("n", "heads", "kv_heads", "head_dim"))
    counts, lens = _lengths(case)
    max_seq = max(lens)
    size, pages, table = _pages(case, g, n, max_seq)
    k_rows, v_rows = (_random_rows(g, pages, kv_heads, size, head_dim) for _ in range(2))
    # heads from flat to peaked
    q = _normal(g, sum(counts), heads, head_dim) * torch.linspace(0.3, 1.5, heads, device="cuda")[:, None]
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    first = [max(0, length - c + 1 - case["window"]) if case["window"] else 0 for c, length in zip(counts, lens)]
    state.update(q=q.to(DTYPES[case["dtype"]]), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                 starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), max_q=max(counts),
                 first=torch.tensor(first, device="cuda"), span=max(a - b for a, b in zip(lens, first)),
                 single=all(c == 1 for c in counts), scale=head_dim ** -0.5)
    _cache(state, n, -(-max_seq // size) * size, kv_heads, head_dim, case["page"], k_rows, v_rows, table)
    return state


def _prepare_sample(case, g, state):
    rows, vocab = case["rows"], case["vocab"]
    # logits of a trained head: a wide bulk and a few tokens far above it, some tokens barred
    logits = 2.0 * _normal(g, rows, vocab)
    logits.scatter_add_(1, torch.randint(0, vocab, (rows, 64), generator=g, device="cuda"), 8 + 3 * _normal(g, rows, 64))
    logits.scatter_(1, torch.randint(0, vocab, (rows, 5), generator=g, device="cuda"), float("-inf"))
    kind = torch.arange(rows, device="cuda") % 6
    full = torch.full((rows,), 1.0, device="cuda")
    temperature, top_p, min_p = 0.8 * full, 0.95 * full, 0.02 * full
    top_k = torch.full((rows,), case["top_k"], dtype=torch.int32, device="cuda")
    if case["filters"] == "none":
        top_p, min_p, top_k = full, 0 * full, 0 * top_k
    elif case["filters"] == "mixed":  # requests of all kinds side by side
        temperature = torch.where(kind == 0, 0.0, torch.where(kind == 1, 1.7, 0.7))
        top_k = torch.where((kind == 2) | (kind == 5), 0, top_k).to(torch.int32)
        top_p = torch.where((kind == 3) | (kind == 5), 1.0, 0.9)
        min_p = torch.where((kind == 4) | (kind == 1), 0.05, 0.0)
    state.update(logits=logits.to(DTYPES[case["dtype"]]), temperature=temperature, top_k=top_k, top_p=top_p,
                 min_p=min_p, u=torch.rand(rows, generator=g, device="cuda"))
    return state


# ---------------------------------------------------------------- one pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    import blocktensor_b200 as bt
    if s["op"] == "norms":
        q, k = bt.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["positions"], s["rope"], eps=s["eps"])
        return {"q": q, "k": k}
    if s["op"] == "append":
        q = s["cache"].append_normed(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["slots"], s["positions"], s["rope"],
                                     eps=s["eps"])
        k, v = s["cache"].read(s["slots"], s["positions"])
        return {"q": q, "k": k, "v": v}
    if s["op"] == "attend":
        return s["cache"].attention(s["q"], s["lens"], q_start=None if s["single"] else s["starts"], max_q=s["max_q"],
                                    window=s["window"], sinks=s["sinks"], scale=s["scale"])
    token, logprob = bt.sample_batch(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    return {"token": token, "logprob": logprob}


def _run_plain(s):
    if s["op"] == "norms":
        return {"q": _normed(s["q"], s["qw"], s).to(s["q"].dtype), "k": _normed(s["k"], s["kw"], s).to(s["k"].dtype)}
    if s["op"] == "append":
        return _plain_append(s)
    return _plain_attend(s) if s["op"] == "attend" else _plain_sample(s)


def _normed(x, weight, s):
    """x / rms(x) * weight of each head, its first `rot` elements rotated in pairs (i, i + rot / 2)."""
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * weight
    half = s["rot"] // 2
    cos, sin = s["rope"][s["positions"].long()][:, None].unbind(-1)
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1)


def _quantise(x):
    """fp32 [..., head_dim] to cache rows."""
    x = torch.nan_to_num(x, nan=0.0).clamp(-LIMIT, LIMIT).unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale, m = ((high - low) / 15).half(), low.half()
    inv = torch.where(scale > 0, 1 / scale.float(), 0.0)
    code = ((x - m.float()) * inv).round().clamp(0, 15).to(torch.uint8).flatten(-2)
    code = code[..., 0::2] | code[..., 1::2] << 4
    return torch.cat([code, torch.cat([scale, m], -1).flatten(-2).view(torch.uint8)], -1)


def _dequantise(rows, head_dim):
    """Cache rows to fp32 [..., head_dim]."""
    code = torch.stack([rows[..., :head_dim // 2] & 15, rows[..., :head_dim // 2] >> 4], -1).flatten(-2)
    scale, low = rows[..., head_dim // 2:].contiguous().view(torch.float16).float().unflatten(-1, (-1, 2)).unbind(-1)
    return (code.unflatten(-1, (-1, GROUP)).float() * scale[..., None] + low[..., None]).flatten(-2)


def _places(s, slots, positions):
    size = s["k_rows"].shape[2]
    return s["table"][slots, positions // size].long(), positions % size


def _plain_append(s):
    page, at = _places(s, s["slots"].long(), s["positions"].long())
    s["k_rows"][page, :, at] = _quantise(_normed(s["k"], s["kw"], s))
    s["v_rows"][page, :, at] = _quantise(s["v"].float())
    k, v = (_dequantise(s[r][page, :, at], s["head_dim"]).half() for r in ("k_rows", "v_rows"))
    return {"q": _normed(s["q"], s["qw"], s).to(s["q"].dtype), "k": k, "v": v}


def _plain_attend(s):
    n, kv_heads, head_dim = s["n"], s["kv_heads"], s["head_dim"]
    lens, starts = s["lens"].long(), s["starts"].long()
    # the positions that some query of a sequence sees: its sinks, then the span up to its length
    sinks = torch.arange(s["sinks"], device="cuda").expand(n, -1)
    span = torch.maximum(s["first"], torch.tensor(s["sinks"], device="cuda"))[:, None] + torch.arange(s["span"], device="cuda")
    at = torch.cat([sinks, span], 1)
    there = at < lens[:, None]
    page, inside = _places(s, torch.arange(n, device="cuda")[:, None], torch.where(there, at, 0))
    k, v = (_dequantise(s[r][page, :, inside], head_dim).transpose(1, 2) for r in ("k_rows", "v_rows"))
    # queries padded to [n][max_q]
    row = starts[:-1, None] + torch.arange(s["max_q"], device="cuda")
    real = row < starts[1:, None]
    q = s["q"][torch.where(real, row, 0)].float().unflatten(2, (kv_heads, -1)).permute(0, 2, 3, 1, 4)
    q_at = lens[:, None] - (starts[1:] - starts[:-1])[:, None] + torch.arange(s["max_q"], device="cuda")
    seen = there[:, None] & (at[:, None] <= q_at[..., None])
    if s["window"]:
        seen &= (at[:, None] > q_at[..., None] - s["window"]) | (at[:, None] < s["sinks"])
    scores = (q.flatten(2, 3) @ k.transpose(-1, -2)).unflatten(2, (-1, s["max_q"])) * s["scale"]
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-38)
    out = (p.flatten(2, 3) @ v).unflatten(2, (-1, s["max_q"])).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[real].to(s["q"].dtype)


def _plain_sample(s):
    x = torch.nan_to_num(s["logits"].float(), nan=float("-inf"), posinf=float("inf"), neginf=float("-inf"))
    greedy = s["temperature"] <= 0
    inv = 1 / torch.where(greedy, 1.0, s["temperature"])[:, None]
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    top = x[:, :1]
    e = torch.where(x == top, 1.0, torch.exp((x - top) * inv))
    weight = (e * UNIT).to(torch.int64)
    rank = torch.arange(x.shape[1], device="cuda")
    # the kept tokens: the top_k largest, of their mass the first top_p, and none below min_p of the largest
    in_k = (s["top_k"][:, None] <= 0) | (rank < s["top_k"][:, None])
    mass = torch.ceil(s["top_p"].double() * (weight * in_k).sum(-1).double()).to(torch.int64)[:, None]
    before = weight.cumsum(-1) - weight
    kept = in_k & (before < mass) & (e >= s["min_p"][:, None]) & ~greedy[:, None] | (rank == 0)
    # the first token in the vocabulary's order whose running sum passes u of the kept mass
    weight = torch.zeros_like(weight).scatter(1, order, weight * kept)
    e = torch.zeros_like(e).scatter(1, order, torch.where(x == top, 0.0, (x - top) * inv))
    running = weight.cumsum(-1)
    total = running[:, -1:]
    target = torch.minimum((s["u"].double()[:, None] * total.double()).to(torch.int64), total - 1)
    token = (running <= target).sum(-1, keepdim=True).clamp(max=x.shape[1] - 1)
    logprob = e.gather(1, token) - torch.log(total.float() / UNIT)
    none = top == float("-inf")  # every token barred
    return {"token": torch.where(none, -1, token)[:, 0].to(torch.int32),
            "logprob": torch.where(none, float("-inf"), logprob)[:, 0]}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    q, k = (_exact_norm(s[x], s[w], s) for x, w in (("q", "qw"), ("k", "kw")))
    if case["op"] == "norms":
        return {"q": q, "k": k}
    return {"q": q, "k": _exact_held(k), "v": _exact_held(s["v"].double())}


def _exact_norm(x, weight, s):
    x = x.double()
    x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + s["eps"]) * weight.double()
    out, half = x.clone(), s["rot"] // 2
    turn = torch.view_as_complex(s["rope"].double().contiguous())[s["positions"].long()][:, None]
    pair = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
    out[..., :half], out[..., half:2 * half] = pair.real, pair.imag
    return out


def _exact_held(x):
    """The values that the 4-bit rows of x stand for."""
    x = x.unflatten(-1, (-1, GROUP))
    low = x.min(-1, keepdim=True).values
    scale = ((x.max(-1, keepdim=True).values - low) / 15).half().double()
    low = low.half().double()
    code = torch.round((x - low) / scale).clamp(0, 15)
    return torch.where(scale > 0, scale * code + low, low).flatten(-2)


def _exact_attend(case, s):
    counts, lens = _lengths(case)
    heads, kv_heads, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if sum(c * length for c, length in zip(counts, lens)) * heads * hd > 3e12:
        return None
    out = torch.zeros(sum(counts), heads, hd, dtype=torch.float64, device="cuda")
    row = 0
    for i, (count, length) in enumerate(zip(counts, lens)):
        at = torch.arange(length, device="cuda")
        q_at = torch.arange(length - count, length, device="cuda")[:, None]
        seen = at <= q_at
        if case["window"]:
            seen &= (q_at - at < case["window"]) | (at < case["sinks"])
        used = seen.any(0).nonzero()[:, 0]
        seen = seen[:, used]
        size = s["k_rows"].shape[2]
        page = s["table"][i, used // size].long()
        for h in range(kv_heads):
            kv = []
            for rows in (s["k_rows"], s["v_rows"]):
                r = rows[page, h, used % size]
                code = torch.empty(len(used), hd, dtype=torch.float64, device="cuda")
                code[:, 0::2], code[:, 1::2] = (r[:, :hd // 2] % 16).double(), (r[:, :hd // 2] // 16).double()
                meta = r[:, hd // 2:].contiguous().view(torch.float16).double()
                kv.append(code * meta[:, 0::2].repeat_interleave(GROUP, 1) + meta[:, 1::2].repeat_interleave(GROUP, 1))
            for head in range(h * heads // kv_heads, (h + 1) * heads // kv_heads):
                t = s["q"][row:row + count, head].double() @ kv[0].T * s["scale"]
                t = torch.softmax(t.masked_fill_(~seen, -math.inf), -1)
                out[row:row + count, head] = t @ kv[1]
        row += count
    return out


def _exact_sample(s):
    """The log-probabilities of the tokens that 64-bit arithmetic draws (the tokens themselves are whole numbers)."""
    got = []
    for b in range(s["logits"].shape[0]):
        x = s["logits"][b].double()
        t, k, p, m = (float(s[f][b]) for f in ("temperature", "top_k", "top_p", "min_p"))
        if t <= 0:
            got.append(0.0)
            continue
        x = (x - x.max()) / t
        value, order = torch.sort(x, dim=0, descending=True, stable=True)
        keep = int(k) if 0 < k < len(x) else len(x)
        w = value.exp()[:keep]
        reach = torch.searchsorted(w.cumsum(0), p * w.sum()) + 1 if p < 1 else keep
        keep = max(1, min(keep, int(reach), int((w >= m).sum())))
        prob = torch.zeros_like(x)
        prob[order[:keep]] = w[:keep] / w[:keep].sum()
        at = torch.searchsorted(prob.cumsum(0), s["u"][b].double(), right=True).clamp(max=len(x) - 1)
        got.append(float(prob[at].log()))
    return {"token": None, "logprob": torch.tensor(got, dtype=torch.float64)}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    if case["op"] == "sample":  # the logits; a difference, a product and an exponential each, and the sums
        return {"bytes": case["rows"] * (case["vocab"] * size + 28), "flops": 4 * case["rows"] * case["vocab"]}
    heads, kv_heads, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] != "attend":
        tokens, rot = case["tokens"], case["rot"]
        q, k = tokens * heads * hd, tokens * kv_heads * hd
        moved = 2 * (q + k) * size + tokens * (rot * 4 + 4) + 2 * hd * 4
        if case["op"] == "append":  # v comes in; k goes to the cache; rows are written, read, and returned in fp16
            moved += tokens * 4 + 4 * tokens * kv_heads * _row_bytes(hd) + 2 * k * 2
        return {"bytes": moved, "flops": 7 * (q + k) + (6 * 2 * k if case["op"] == "append" else 0)}
    pairs = rows = 0
    counts, lens = _lengths(case)
    for c, length in zip(counts, lens):
        if not case["window"]:
            pairs += c * length - c * (c - 1) // 2
            rows += length
            continue
        w, sinks = case["window"], case["sinks"]
        pairs += sum(min(p + 1, w) + min(sinks, max(0, p + 1 - w)) for p in range(length - c, length))
        lo = max(0, length - c + 1 - w)
        rows += length - lo + min(sinks, lo)
    return {"bytes": rows * kv_heads * 2 * _row_bytes(hd) + 2 * sum(counts) * heads * hd * size,
            "flops": 4 * hd * heads * pairs}
