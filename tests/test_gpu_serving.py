"""GPU: the serving operators against plain 64-bit implementations.

Tolerances, from the arithmetic and not from runs:

* norms: fp32 throughout: the mean of squares (a tree over head_dim terms, at most 12 roundings of 2^-24),
  rsqrt (2 ulp), two products, the rotation's two products and a sum: within 2^-19 of |a| + |b|, the pair's
  magnitudes, plus the result's own rounding (half an ulp of its type).
* the cache's codes are exact for given keys and values: the same fp32 steps, compared as equal.
* attention: a score of terms q_i k_i carries at most 2^-19 of sum |q_i k_i| in the fp32 forms, and 6 standard
  deviations of independent 2^-11 roundings, 6 * 2^-11 * sqrt(sum (q_i k_i)^2), where operands are held in fp16
  (16-bit types); probabilities 2^-18 or 4 * 2^-11 alike; all of it relative to the largest |v|.
* sampling: whole-number weights of fp32 exponentials, each within 2^-21 of itself (exp's 2 ulp and the fp32
  argument's rounding at |x| <= 28): a draw u within 2^-20 of a boundary between two tokens may fall either
  way, and a cut within 2^-20 of its mass may; test inputs whose 64-bit margins are smaller are not judged by
  equality (their count is bounded).
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DT = ["float32", "float16", "bfloat16"]
HALF_ULP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}  # relative, generous by up to 2
TINY = {"float32": 1e-37, "float16": 2.0 ** -24, "bfloat16": 1e-37}


def T():
    import torch
    return torch


def gen(seed):
    return T().Generator("cuda").manual_seed(seed)


def randn(g, *shape):
    return T().randn(*shape, generator=g, device="cuda")


def ints(values):
    return T().tensor(values, dtype=T().int32, device="cuda")


# ---------------------------------------------------------------- norms

def ref_norm_rope(x, w, eps, pos, table):
    """(result, |a| + |b| of every pair) in float64; w None: no norm, table None: no rotation."""
    torch = T()
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    out, mag = x.clone(), x.abs().clone()
    if table is not None:
        h = table.shape[1]
        c, s = (table[pos.long()].double()[:, None, :, i] for i in (0, 1))
        a, b = x[..., :h], x[..., h:2 * h]
        out[..., :h], out[..., h:2 * h] = a * c - b * s, b * c + a * s
        mag[..., :h] = mag[..., h:2 * h] = a.abs() + b.abs()
    return out, mag


def close_norm(got, want, mag, dt):
    err = (got.double() - want).abs()
    tol = 2.0 ** -19 * mag + HALF_ULP[dt] * want.abs() + TINY[dt]
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("tokens,heads,kv,hd,rot", [
    (1, 1, 1, 64, 64), (1, 32, 32, 128, 128), (3, 5, 1, 256, 256), (7, 12, 4, 128, 64), (257, 8, 2, 64, 16), (601, 3, 3, 128, 112),
    (2, 71, 9, 256, 96)])
def test_norm_rope(cuda, dt, tokens, heads, kv, hd, rot):
    torch = T()
    g = gen(tokens * 1000 + heads)
    dtype = getattr(torch, dt)
    qkv = (randn(g, tokens, heads + 2 * kv, hd) * 3).to(dtype)
    q, k = qkv[:, :heads], qkv[:, heads:heads + kv]
    w = 1 + 0.3 * randn(g, 2, hd)
    table = cuda.rope_table(700, rot, 500000.0)
    pos = torch.randint(0, 700, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    qo, ko = cuda.qk_norm_rope(q, k, w[0], w[1], pos, table, eps=1e-5)
    assert qo.dtype == dtype and qo.is_contiguous() and qo.shape == q.shape
    close_norm(qo, *ref_norm_rope(q, w[0], 1e-5, pos, table), dt)
    close_norm(ko, *ref_norm_rope(k, w[1], 1e-5, pos, table), dt)
    # in place, on the fused buffer; queries alone; no norm; no rotation: the same values
    keep = qkv.clone()
    a, b = cuda.qk_norm_rope(q, k, w[0], w[1], pos, table, eps=1e-5, q_out=q, k_out=k)
    assert a is q and torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(qkv[:, heads + kv:], keep[:, heads + kv:])
    q = keep[:, :heads]
    assert torch.equal(cuda.qk_norm_rope(q, None, w[0], None, pos, table)[0], qo)
    close_norm(cuda.qk_norm_rope(q, None, None, None, pos, table)[0], *ref_norm_rope(q, None, 0, pos, table), dt)
    close_norm(cuda.qk_norm_rope(q, None, w[0], None, pos, None)[0], *ref_norm_rope(q, w[0], 1e-5, pos, None), dt)


@pytest.mark.parametrize("dt", DT)
def test_norm_rope_unaligned_and_head_major(cuda, dt):
    """Data one element off a 16-byte boundary, and a [heads][tokens] layout."""
    torch = T()
    g = gen(5)
    dtype = getattr(torch, dt)
    w = 1 + 0.3 * randn(g, 2, 128)
    table, pos = cuda.rope_table(64, 128), ints([63, 0, 5, 1])
    flat = randn(g, 4 * 6 * 128 + 1).to(dtype)
    off = flat[1:].view(4, 6, 128)
    major = randn(g, 6, 4, 128).to(dtype).transpose(0, 1)
    for x in (off, major):
        q, k = x[:, :4], x[:, 4:]
        qo, ko = cuda.qk_norm_rope(q, k, w[0], w[1], pos, table)
        close_norm(qo, *ref_norm_rope(q, w[0], 1e-5, pos, table), dt)
        close_norm(ko, *ref_norm_rope(k, w[1], 1e-5, pos, table), dt)


def test_norm_rope_edges(cuda):
    """A zero row, a huge one, NaN and infinity stay in their own rows; a position outside the table gives NaN."""
    torch = T()
    w, table = torch.ones(64, device="cuda"), cuda.rope_table(8, 64)
    q = torch.ones(5, 2, 64, device="cuda")
    q[0, 0] = 0
    q[1, 0] = 1e18
    q[2, 0, 7] = float("nan")
    out, _ = cuda.qk_norm_rope(q, None, w, None, ints([0, 1, 2, 8, -1]), table)
    assert bool((out[0, 0] == 0).all()) and bool(out[1].isfinite().all()) and bool(out[2, 0].isnan().all())
    assert bool(out[2, 1].isfinite().all()) and bool(out[3:].isnan().all())
    empty, _ = cuda.qk_norm_rope(q[:0], None, w, None, ints([]), table)
    assert empty.shape == (0, 2, 64)


# ---------------------------------------------------------------- cache rows

def ref_rows(x):
    """[..., hd] (any type) to the rows bt_kv4 describes, with the same fp32 steps in numpy."""
    x = np.nan_to_num(x.float().cpu().numpy(), nan=0.0, posinf=57344.0, neginf=-57344.0).clip(-57344, 57344).astype(np.float32)
    s = x.shape
    x = x.reshape(*s[:-1], s[-1] // 64, 64)
    lo, hi = x.min(-1), x.max(-1)
    scale, low = ((hi - lo) * (np.float32(1) / np.float32(15))).astype(np.float16), lo.astype(np.float16)
    sf = scale.astype(np.float32)
    inv = np.where(sf > 0, np.float32(1) / np.where(sf > 0, sf, np.float32(1)), np.float32(0)).astype(np.float32)
    code = np.rint((x - low.astype(np.float32)[..., None]) * inv[..., None]).clip(0, 15).astype(np.uint8).reshape(s)
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    meta = np.stack([scale, low], -1).reshape(*s[:-1], -1).view(np.uint8)
    return np.concatenate([packed, meta], -1)


def ref_values(rows, hd):
    """Rows (uint8 tensor [..., row]) to float64 values."""
    torch = T()
    code = torch.empty(*rows.shape[:-1], hd, dtype=torch.float64, device=rows.device)
    code[..., 0::2], code[..., 1::2] = (rows[..., :hd // 2] & 15).double(), (rows[..., :hd // 2] >> 4).double()
    meta = rows[..., hd // 2:].contiguous().view(torch.float16).double()
    return code * meta[..., 0::2].repeat_interleave(64, -1) + meta[..., 1::2].repeat_interleave(64, -1)


def edge_rows(g, *shape):
    """Normal rows with constant, zero, tiny, huge, infinite and NaN groups among them."""
    x = randn(g, *shape)
    flat = x.view(-1, 64)
    n = flat.shape[0]
    for i, v in enumerate((0.0, 2.5, -1e-7, 1e-9, 3e38, float("inf"), float("nan"))):
        if i < n:
            flat[(i * 5) % n, : 64 if i % 2 else 11] = v
    if n > 40:
        flat[37] *= 1e4
        flat[38] *= 1e-6
        flat[39, 3] = -float("inf")
    return x


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("hd,kv,page", [(64, 1, 0), (64, 3, 16), (128, 2, 64), (256, 1, 0), (128, 8, 256)])
def test_append_and_read(cuda, dt, hd, kv, page):
    torch = T()
    g = gen(hd + kv + page)
    n_seq, max_seq, tokens = 5, 211, 97
    cache = cuda.KV4Cache(n_seq, max_seq, kv, hd, page_tokens=page, n_pages=80 if page == 16 else 20)
    if page:
        for s in (3, 0, 4, 1, 2):
            cache.reserve(s, max_seq)
    k, v = (edge_rows(g, tokens, kv, hd).to(getattr(torch, dt)) for _ in range(2))
    flat = torch.randperm(n_seq * max_seq, generator=g, device="cuda")[:tokens]
    slots, pos = (flat // max_seq).int(), (flat % max_seq).int()
    cache.append(k, v, slots, pos)
    cache.check()
    at = (slots.long(), pos.long())
    pages = cache.page_table[at[0], at[1] // page].long() if page else at[0]
    inside = at[1] % cache.page_tokens
    for rows, x in ((cache.k_rows, k), (cache.v_rows, v)):
        assert np.array_equal(rows[pages, :, inside].cpu().numpy(), ref_rows(x))
    # every other row is as it was
    cache.k_rows[pages, :, inside] = 0
    cache.v_rows[pages, :, inside] = 0
    assert int(cache.k_rows.max()) == 0 and int(cache.v_rows.max()) == 0
    cache.append(k, v, slots, pos)
    for out in DT:
        rk, rv = cache.read(slots, pos, dtype=getattr(torch, out))
        for r, x in ((rk, cache.k_rows), (rv, cache.v_rows)):
            want = ref_values(x[pages, :, inside], hd)
            fin = want.abs() < 65000
            err = (r.double() - want).abs()[fin]
            assert bool((err <= (HALF_ULP[out] + 2.0 ** -23) * (want.abs()[fin] + 57344 * 2.0 ** -24) + TINY[out]).all())


def test_append_ranges(cuda):
    """Slots, positions and pages out of range store nothing and are reported; padding is skipped quietly."""
    torch = T()
    cache = cuda.KV4Cache(2, 40, 1, 64, page_tokens=16, n_pages=4)
    cache.reserve(0, 40)
    x = torch.ones(1, 1, 64, device="cuda")
    for slot, pos in ((2, 0), (0, 40), (0, -1), (1, 0)):
        cache.append(x, x, ints([slot]), ints([pos]))
        with pytest.raises(IndexError):
            cache.check()
        k, _ = cache.read(ints([slot]), ints([pos]))
        assert bool((k == 0).all())
        with pytest.raises(IndexError):
            cache.check()
    cache.page_table[1, 0] = 4
    cache.append(x, x, ints([1]), ints([3]))
    with pytest.raises(IndexError):
        cache.check()
    cache.append(x, x, ints([-1]), ints([3]))
    cache.check()
    assert int(cache.k_rows.max()) == 0 and int(cache.v_rows.max()) == 0
    cache.append(x[:0], x[:0], ints([]), ints([]))


@pytest.mark.parametrize("dt", DT)
def test_append_normed(cuda, dt):
    """The queries are qk_norm_rope's, bit for bit, and the rows are those of its keys in fp32."""
    torch = T()
    g = gen(3)
    dtype = getattr(torch, dt)
    tokens, heads, kv, hd = 33, 6, 2, 128
    qkv = randn(g, tokens, heads + 2 * kv, hd).to(dtype)
    q, k, v = qkv.split([heads, kv, kv], 1)
    w = 1 + 0.3 * randn(g, 2, hd)
    table = cuda.rope_table(64, hd)
    pos, slots = torch.arange(5, 5 + tokens, dtype=torch.int32, device="cuda"), torch.ones(tokens, dtype=torch.int32, device="cuda")
    cache = cuda.KV4Cache(2, 40, kv, hd)
    qo = cache.append_normed(q, k, v, w[0], w[1], slots, pos, table)
    want_q, _ = cuda.qk_norm_rope(q, k, w[0], w[1], pos, table)
    assert torch.equal(qo, want_q)
    _, k32 = cuda.qk_norm_rope(q.float(), k.float(), w[0], w[1], pos, table)
    assert np.array_equal(cache.k_rows[1, :, 5:5 + tokens].transpose(0, 1).cpu().numpy(), ref_rows(k32))
    assert np.array_equal(cache.v_rows[1, :, 5:5 + tokens].transpose(0, 1).cpu().numpy(), ref_rows(v))
    # keys and values alone
    only = cuda.KV4Cache(2, 40, kv, hd)
    assert only._append(None, k, v, None, w[1], slots, pos, table, 1e-5, None, None) is None
    assert torch.equal(only.k_rows, cache.k_rows)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_append_normed_plain_codes(cuda, dt, hd):
    """The cached rows are those of keys that plain fp32 PyTorch norms and rotates, bit for bit (a code at the
    edge between two steps would fall either way with the last bit of the norm)."""
    torch = T()
    g = gen(hd)
    dtype = getattr(torch, dt)
    tokens, kv = 3001, 4
    k, v = ((randn(g, tokens, kv, hd) * (1 + 2 * torch.rand(hd, generator=g, device="cuda"))).to(dtype) for _ in range(2))
    w = 1 + 0.3 * randn(g, hd)
    table = cuda.rope_table(tokens, hd, 500000.0)
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda")
    cache = cuda.KV4Cache(1, tokens, kv, hd)
    cache._append(None, k, v, None, w, torch.zeros_like(pos), pos, table, 1e-5, None, None)
    x = k.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w
    c, s = table[:, None, :, 0], table[:, None, :, 1]
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    want = ref_rows(torch.cat([a * c - b * s, a * s + b * c], -1))
    assert np.array_equal(cache.k_rows[0, :, :tokens].transpose(0, 1).cpu().numpy(), want)


# ---------------------------------------------------------------- attention

class Case:
    """Sequences with random cache rows, garbage wherever no query may look."""

    def __init__(self, cuda, seed, dt, hd, kv, group, lens, counts, page=0, window=0, sinks=0, shuffle=False, spread=1.0,
                 layout="plain"):
        torch = T()
        g = gen(seed)
        self.dt, self.hd, self.kv, self.group, self.lens, self.counts = dt, hd, kv, group, lens, counts
        self.window, self.sinks = window, sinks
        n, heads = len(lens), kv * group
        max_seq = max(max(lens), 1) + 3
        n_slots = n + (2 if shuffle else 0)
        cache = cuda.KV4Cache(n_slots, max_seq, kv, hd, page_tokens=page, n_pages=n_slots * -(-max_seq // page) if page else 0,
                              page_table=None)
        if page:
            order = torch.randperm(cache.n_pages, generator=g, device="cuda").int()
            cache.page_table[:] = order.view(n_slots, -1)
        self.cache = cache
        self.slots = torch.randperm(n_slots, generator=g, device="cuda")[:n].int() if shuffle else None
        for rows in (cache.k_rows, cache.v_rows):
            rows.fill_(0xFF)  # NaN scales and mins
        self.k, self.v = [], []
        slot_of = self.slots.tolist() if shuffle else range(n)
        for i, length in enumerate(lens):
            pos = torch.arange(length, device="cuda")
            k, v = (randn(g, length, kv, hd) * spread for _ in range(2))
            seen = torch.zeros(length, dtype=torch.bool, device="cuda")
            first = max(0, length - counts[i])
            lo = max(0, first - window + 1) if window else 0
            if counts[i]:
                seen[lo:] = True
                seen[:min(sinks, length) if window else 0] = True
            live = pos[seen]
            s = torch.full((len(live),), slot_of[i], dtype=torch.int32, device="cuda")
            if len(live):
                cache.append(k[seen], v[seen], s, live.int())
            page_of = cache.page_table[slot_of[i], live // page].long() if page else s.long()
            if page:  # pages that nobody looks at need not be there
                gone = torch.ones(cache.max_pages, dtype=torch.bool, device="cuda")
                gone[live // page] = False
                cache.page_table[slot_of[i]][gone] = -1
            vals = []
            for rows in (cache.k_rows, cache.v_rows):
                full = torch.zeros(length, kv, hd, dtype=torch.float64, device="cuda")
                if len(live):
                    full[seen] = ref_values(rows[page_of, :, live % cache.page_tokens], hd)
                vals.append(full)
            self.k.append(vals[0])
            self.v.append(vals[1])
        total = sum(counts)
        dtype = getattr(torch, dt)
        q = randn(g, total, heads, hd) * torch.linspace(0.2, 2.0, heads, device="cuda")[:, None]
        if layout == "plain":
            self.q = q.to(dtype)
        elif layout == "fused":  # a slice of a wider buffer
            wide = torch.zeros(total, heads + 3, hd, dtype=dtype, device="cuda")
            wide[:, 1:1 + heads] = q.to(dtype)
            self.q = wide[:, 1:1 + heads]
        else:  # one element off alignment
            flat = torch.zeros(total * heads * hd + 1, dtype=dtype, device="cuda")
            self.q = flat[1:].view(total, heads, hd)
            self.q.copy_(q)
        self.scale = hd ** -0.5
        self.starts = ints(np.concatenate([[0], np.cumsum(counts)]).tolist())

    def run(self, **kw):
        single = all(c == 1 for c in self.counts)
        args = dict(q_start=None if single else self.starts, slots=self.slots, window=self.window, sinks=self.sinks,
                    max_q=max(self.counts) if self.counts else 0)
        args.update(kw)
        out = self.cache.attention(self.q, ints(self.lens), **args)
        self.cache.check()
        return out

    def want(self):
        """(values, tolerance) in float64."""
        torch = T()
        heads, hd = self.kv * self.group, self.hd
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(out)
        row = 0
        for i, (length, count) in enumerate(zip(self.lens, self.counts)):
            at, q_at = torch.arange(length, device="cuda"), torch.arange(length - count, length, device="cuda")[:, None]
            seen = (at <= q_at)
            if self.window:
                seen &= (at > q_at - self.window) | (at < self.sinks)
            for h in range(heads):
                k, v = self.k[i][:, h // self.group], self.v[i][:, h // self.group]
                q = self.q[row:row + count, h].double() * self.scale
                s = (q @ k.T).masked_fill(~seen, -math.inf)
                p = torch.nan_to_num(torch.softmax(s, -1)) if length else s
                o = p @ v
                out[row:row + count, h] = o
                if length == 0 or count == 0:
                    continue
                big = v.abs().max()
                if self.dt == "float32":
                    mag = ((q.abs() @ k.abs().T) * seen).amax(-1, keepdim=True)
                    t = (mag * 2.0 ** -19 + 2.0 ** -18) * big
                else:
                    mag = ((q.pow(2) @ k.pow(2).T) * seen).amax(-1, keepdim=True).sqrt()
                    t = (6 * mag + 4) * 2.0 ** -11 * big + HALF_ULP[self.dt] * o.abs()
                tol[row:row + count, h] = t.expand_as(o)
            row += count
        return out, tol

    def check(self, **kw):
        got = self.run(**kw)
        want, tol = self.want()
        assert got.dtype == self.q.dtype and got.shape == self.q.shape
        err = (got.double() - want).abs()
        assert bool((err <= tol).all()), f"off by {float((err / tol.clamp(min=1e-30)).max()):.3g} tolerances"
        return got


SINGLE = [
    # lens, kv, group, page, window, sinks
    ([1], 1, 1, 0, 0, 0),
    ([0], 1, 3, 0, 0, 0),
    ([550], 4, 1, 0, 0, 0),
    ([15, 16, 17, 0, 1], 2, 8, 16, 0, 0),
    ([700, 33, 129, 64, 255], 2, 4, 64, 0, 0),
    ([1000, 5, 260], 1, 12, 32, 0, 0),
    ([2049], 8, 5, 1024, 0, 0),
    ([900, 3, 400, 40, 0], 2, 8, 16, 100, 4),
    ([900, 120], 3, 2, 0, 1, 0),
    ([333, 7, 50], 1, 9, 16, 17, 37),
    ([500], 2, 16, 64, 10000, 5),
    ([64] * 70, 1, 8, 16, 0, 0),
]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("i", range(len(SINGLE)))
def test_attention_single(cuda, dt, hd, i):
    lens, kv, group, page, window, sinks = SINGLE[i]
    Case(cuda, 100 + i, dt, hd, kv, group, lens, [1] * len(lens), page, window, sinks, shuffle=i % 2 == 1,
         layout=["plain", "fused", "off"][i % 3]).check()


DEALT = [  # items around the numbers of SMs and of half of them, even and ragged
    ([900] * 9, 8, 8),
    ([129] * 16, 8, 3),
    ([60, 4000, 31, 1, 0, 700, 33, 32, 64, 65], 12, 1),
    ([2500] + [3] * 72, 2, 4),
    ([33] * 147, 1, 1),
    ([70, 1] * 74, 1, 2),
    ([40] * 149, 1, 2),
    ([0] * 200 + [500, 20], 4, 1),
]


@pytest.mark.parametrize("dt,hd", [("float32", 64), ("float16", 128), ("bfloat16", 256)])
@pytest.mark.parametrize("i", range(len(DEALT)))
def test_attention_dealing(cuda, dt, hd, i):
    lens, kv, group = DEALT[i]
    Case(cuda, 300 + i, dt, hd, kv, group, lens, [1] * len(lens), page=16 * (i % 2)).check()


CHUNKS = [
    # lens, counts, kv, group, page, window, sinks
    ([2], [2], 1, 1, 0, 0, 0),
    ([1, 7, 0, 64], [1, 7, 0, 64], 2, 4, 16, 0, 0),
    ([300], [300], 1, 8, 0, 0, 0),
    ([300, 513], [17, 1], 2, 1, 64, 0, 0),
    ([129, 700, 128, 31], [128, 200, 127, 31], 2, 3, 32, 0, 0),
    ([800], [260], 1, 12, 128, 50, 4),
    ([260, 20, 400], [260, 20, 5], 2, 8, 16, 33, 70),
    ([1100], [600], 4, 8, 256, 400, 1),
    ([5, 40], [9, 3], 1, 5, 16, 0, 0),  # more queries than positions: the first rows see nothing
    ([600], [600], 1, 16, 0, 1, 0),
]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("i", range(len(CHUNKS)))
def test_attention_chunks(cuda, dt, hd, i):
    lens, counts, kv, group, page, window, sinks = CHUNKS[i]
    Case(cuda, 200 + i, dt, hd, kv, group, lens, counts, page, window, sinks, shuffle=i % 2 == 0,
         layout=["plain", "fused", "off"][i % 3]).check()


def test_attention_empty_rows_are_zero(cuda):
    c = Case(cuda, 7, "float16", 128, 1, 4, [3, 0], [5, 2])
    got = c.run()
    assert bool((got[:2] == 0).all()) and bool((got[5:] == 0).all()) and bool((got[2:5] != 0).any())


@pytest.mark.parametrize("dt", DT)
def test_attention_magnitudes(cuda, dt):
    """Large and tiny keys and values, peaked scores, constant values."""
    for spread in (1e-4, 30.0):
        Case(cuda, 11, dt, 128, 2, 4, [400, 90], [1, 1], 16, spread=spread).check()
        Case(cuda, 12, dt, 64, 1, 4, [400, 90], [40, 90], 16, spread=spread).check()


@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 80, 200]])
def test_attention_repeats_and_neighbours(cuda, counts):
    """The same bits again, whatever ran before on the workspace; a sequence's rows do not depend on what
    runs beside it beyond rounding; max_q not known gives the same values."""
    torch = T()
    c = Case(cuda, 21, "float16", 128, 2, 4, [700, 90, 300], counts, 16)
    first = c.check()
    Case(cuda, 22, "float16", 128, 2, 4, [900] * 5, [1] * 5, 64).run()
    assert torch.equal(first, c.run())
    c.check(max_q=0)


def test_attention_streams_and_out(cuda):
    """On another stream, into a strided output, while the current stream is busy."""
    torch = T()
    c = Case(cuda, 31, "bfloat16", 128, 2, 4, [600, 77], [1, 1], 64)
    want, tol = c.want()
    side = torch.cuda.Stream()
    wide = torch.full((2, 12, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    lens = ints(c.lens)
    side.wait_stream(torch.cuda.current_stream())
    out = c.cache.attention(c.q, lens, out=wide[:, 2:10], stream=side)
    side.synchronize()
    assert bool(((out.double() - want).abs() <= tol).all())
    assert bool((wide[:, :2] == 7).all()) and bool((wide[:, 10:] == 7).all())
    with torch.cuda.stream(side):
        again = c.cache.attention(c.q, lens)
    side.synchronize()
    assert torch.equal(again, out)


def test_attention_in_a_graph(cuda):
    """Captured once, replayed with other lengths."""
    torch = T()
    c = Case(cuda, 41, "float16", 64, 2, 8, [500, 300], [1, 1], 16)
    lens = ints([500, 300])
    out = torch.empty_like(c.q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.cache.attention(c.q, lens, out=out)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.cache.attention(c.q, lens, out=out)
    for new in ([500, 300], [17, 1], [499, 0]):
        lens.copy_(ints(new))
        graph.replay()
        torch.cuda.synchronize()
        c.lens = new
        d = [x[:n] for x, n in zip(c.k, new)], [x[:n] for x, n in zip(c.v, new)]
        keep, (c.k, c.v) = (c.k, c.v), d
        want, tol = c.want()
        c.k, c.v = keep
        assert bool(((out.double() - want).abs() <= tol).all())


def test_attention_ranges(cuda):
    """Lengths, slots and pages out of range are reported and never followed."""
    torch = T()
    c = Case(cuda, 51, "float16", 64, 1, 2, [40, 20], [1, 1], 16)
    for lens, slots in (([44, 20], None), ([-1, 20], None), ([40, 20], [0, 2]), ([40, 20], [-1, 1])):
        c.cache.attention(c.q, ints(lens), slots=None if slots is None else ints(slots))
        with pytest.raises(IndexError):
            c.cache.check()
    c.cache.page_table[0, 1] = 1000
    out = c.cache.attention(c.q, ints([40, 20]))
    with pytest.raises(IndexError):
        c.cache.check()
    want, tol = c.want()
    assert bool(((out[1].double() - want[1]).abs() <= tol[1]).all()) and bool(out.isfinite().all())


def test_attention_past_4gb(cuda):
    """Rows beyond the first 4 GB of the pool."""
    torch = T()
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    g = gen(61)
    kv, hd, max_seq = 4, 256, 2_200_000  # 144 B * 4 * 2.2 M = 1.27 GB a slot, 5 slots a side
    cache = cuda.KV4Cache(5, max_seq, kv, hd)
    length = 2_100_000
    window = 300
    pos = torch.arange(length - window, length, device="cuda").int()
    k, v = randn(g, window, kv, hd), randn(g, window, kv, hd)
    cache.append(k, v, torch.full_like(pos, 4), pos)
    q = randn(g, 1, kv, hd).half()
    out = cache.attention(q, ints([length]), slots=ints([4]), window=window)
    cache.check()
    kk, vv = (ref_values(r[4, :, length - window:length], hd) for r in (cache.k_rows, cache.v_rows))
    p = torch.softmax(torch.einsum("hd,hjd->hj", q[0].double() / 16, kk), -1)
    want = torch.einsum("hj,hjd->hd", p, vv)
    assert float((out[0].double() - want).abs().max()) <= (6 * 1.0 + 4) * 2.0 ** -11 * float(vv.abs().max())


# ---------------------------------------------------------------- sampling

def ref_sample(x, t, k, p, mp, u):
    """(token, logprob, margin) of one row in float64: margin is u's and the cuts' distance from where the
    result changes."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    m = x.max()
    if m == -np.inf:
        return -1, -np.inf, 1.0
    order = np.argsort(-x, kind="stable")
    if t <= 0:
        return int(order[0]), 0.0, 1.0
    with np.errstate(invalid="ignore"):
        e = np.where(x == m, 1.0, np.exp((x - m) / t))
    e = np.floor(e * 2.0 ** 40) / 2.0 ** 40
    keep = k if 0 < k < len(x) else len(x)
    margin = 1.0
    if p < 1:
        c = np.cumsum(e[order[:keep]])
        want = p * c[-1]
        margin = min(margin, np.abs(c - want).min() / c[-1])
        keep = min(keep, int(np.searchsorted(c, want)) + 1)
    if mp > 0:
        ok = e[order[:keep]] >= mp
        margin = min(margin, np.abs(e[order[:keep]] - mp).min())
        keep = max(1, int(ok.sum()))
    w = np.zeros(len(x))
    w[order[:keep]] = e[order[:keep]]
    c = np.cumsum(w)
    at = min(max(u, 0.0), 1 - 2.0 ** -25) * c[-1]
    margin = min(margin, np.abs(c[w > 0] - at).min() / c[-1])
    token = int(np.searchsorted(c, at, side="right"))
    return token, (0.0 if x[token] == m else (x[token] - m) / t) - math.log(c[-1]), margin


def check_rows(cuda, logits, u, t, k, p, mp, exact=False):
    torch = T()
    dev = lambda a, d: torch.tensor(a, dtype=d, device="cuda")  # noqa: E731
    tok, lp = cuda.sample_batch(logits, dev(u, torch.float32), dev(t, torch.float32), dev(k, torch.int32), dev(p, torch.float32),
                                dev(mp, torch.float32))
    tok2, lp2 = cuda.sample_batch(logits, dev(u, torch.float32), dev(t, torch.float32), dev(k, torch.int32),
                                  dev(p, torch.float32), dev(mp, torch.float32))
    assert torch.equal(tok, tok2) and torch.equal(lp, lp2)
    x = logits.float().cpu().numpy()
    tok, lp, close = tok.tolist(), lp.tolist(), 0
    f = lambda v: float(np.float32(v))  # noqa: E731
    for b in range(len(tok)):
        want, want_lp, margin = ref_sample(x[b], f(t[b]), k[b], f(p[b]), f(mp[b]), f(u[b]))
        if margin < 2.0 ** -20 and not exact:
            close += tok[b] != want
            continue
        assert tok[b] == want, (b, tok[b], want, margin)
        # the fp32 argument's rounding at |x| <= 28 and the log's: 2^-19
        assert lp[b] == want_lp or abs(lp[b] - want_lp) <= 2.0 ** -19, (b, lp[b], want_lp)
    return close


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("vocab", [1, 2, 37, 1000, 4096, 16385, 32000, 50257, 128256, 200001, 300007])
def test_sample(cuda, dt, vocab):
    """Rows with every kind of parameters side by side; vocabularies of one to eight CTAs a row and beyond."""
    torch = T()
    rng = np.random.default_rng(vocab)
    rows = 24
    g = gen(vocab)
    logits = randn(g, rows, vocab) * 2
    logits[:, :: max(1, vocab // 50)] += 6
    logits = logits.to(getattr(torch, dt))  # 16-bit types: many equal logits
    t = [[1.0, 0.7, 0.0, 1.9, 0.05][i % 5] for i in range(rows)]
    k = [[0, 1, 50, vocab, 1000, 7, -3][i % 7] for i in range(rows)]
    p = [[1.0, 0.9, 0.5, 0.999, 0.0, 1.5][i % 6] for i in range(rows)]
    mp = [[0.0, 0.05, 0.0, 0.0, 1.0, 0.5, 1.5][(i // 2) % 7] for i in range(rows)]
    u = [0.0, 0.9999999] + rng.random(rows - 2).astype(np.float32).tolist()
    assert check_rows(cuda, logits, u, t, k, p, mp) <= 4


@pytest.mark.parametrize("vocab", [600, 40000, 300000])
def test_sample_equal_logits(cuda, vocab):
    """Ties: the lowest ids are kept, and the draw counts through them exactly."""
    torch = T()
    rows = 8
    logits = torch.zeros(rows, vocab, device="cuda")
    logits[4:, vocab // 3: vocab // 2] = 1.0
    n = vocab // 2 - vocab // 3
    k = [0, vocab // 2, 1, 5, 0, n, n + 7, 3]
    p = [1.0, 1.0, 1.0, 0.4, 0.5, 1.0, 0.9, 1.0]
    u = [0.0, 0.999, 0.5, 0.9, 0.3, 0.7, 0.2, 0.95]
    assert check_rows(cuda, logits, u, [1.0] * rows, k, p, [0.0] * rows) == 0


def test_sample_barred(cuda):
    """-inf and NaN logits are never drawn; a row of nothing else gives -1; +inf takes everything; -0 equals 0."""
    torch = T()
    inf, nan = float("inf"), float("nan")
    x = torch.full((9, 5000), -inf, device="cuda")
    x[1, 77] = -5.0
    x[2, 9] = nan
    x[3] = 0.0
    x[3, ::2] = nan
    x[4, [5, 6]] = inf
    x[4, 7] = 3.0
    x[5] = -3e38
    x[6, 3], x[6, 4] = -0.0, 0.0
    x[7] = 1.0
    x[8, 4999] = 2.0
    u = torch.tensor([0.5, 0.9, 0.1, 0.0, 0.7, 0.5, 0.0, 0.999999, 0.0], device="cuda")
    tok, lp = cuda.sample_batch(x, u)
    assert tok.tolist()[:5] == [-1, 77, -1, 1, 6] and lp[0] == -inf and lp[2] == -inf
    assert tok.tolist()[5:] == [2500, 3, 4999, 4999]
    ones = torch.ones(9, dtype=torch.int32, device="cuda")
    tok, lp = cuda.sample_batch(x, u, top_k=ones)
    assert tok.tolist() == [-1, 77, -1, 1, 5, 0, 3, 0, 4999] and lp[4] == 0
    tok, _ = cuda.sample_batch(x, u, temperature=torch.zeros(9, device="cuda"))
    assert tok.tolist() == [-1, 77, -1, 1, 5, 0, 3, 0, 4999]


def test_sample_strides(cuda):
    """Rows of a wider buffer, at any alignment."""
    torch = T()
    g = gen(71)
    for dt in DT:
        for off in (0, 1, 3):
            buf = randn(g, 6, 2100).to(getattr(torch, dt))
            x = buf[:, off:off + 2000 + off]
            assert check_rows(cuda, x, [0.1, 0.3, 0.5, 0.7, 0.9, 0.95], [0.8] * 6, [40] * 6, [0.95] * 6, [0.01] * 6) <= 1


def test_sample_distribution(cuda):
    """Over evenly spaced u the draws have the probabilities of the kept tokens."""
    torch = T()
    n = 4096
    x = torch.tensor([0.0, 1.0, 2.0, -1.0, 3.0], device="cuda").expand(n, 5).contiguous()
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tok, _ = cuda.sample_batch(x, u, top_k=torch.full((n,), 3, dtype=torch.int32, device="cuda"))
    got = torch.bincount(tok.long(), minlength=5).double().cpu() / n
    e = torch.tensor([0.0, math.e, math.e ** 2, 0.0, math.e ** 3], dtype=torch.float64)
    assert float((got - e / e.sum()).abs().max()) <= 1.0 / n


def test_refusals_on_tensors(cuda):
    torch = T()
    q = torch.zeros(2, 4, 128, device="cuda")
    w, pos, table = torch.ones(128, device="cuda"), ints([0, 1]), cuda.rope_table(4, 128)
    cache = cuda.KV4Cache(2, 32, 2, 128)
    bad = [
        lambda: cuda.qk_norm_rope(q.double(), None, w, None, pos, table),
        lambda: cuda.qk_norm_rope(q.cpu(), None, w, None, pos, table),
        lambda: cuda.qk_norm_rope(q[0], None, w, None, pos, table),
        lambda: cuda.qk_norm_rope(q.transpose(1, 2), None, w, None, pos, table),
        lambda: cuda.qk_norm_rope(q, q[:1], w, w, pos, table),
        lambda: cuda.qk_norm_rope(q, None, w.half(), None, pos, table),
        lambda: cuda.qk_norm_rope(q, None, w[:64], None, pos, table),
        lambda: cuda.qk_norm_rope(q, None, w, None, pos.long(), table),
        lambda: cuda.qk_norm_rope(q, None, w, None, pos, table.half()),
        lambda: cuda.qk_norm_rope(q, None, w, None, pos, table, q_out=q.half()),
        lambda: cache.append(q, q, pos, pos),
        lambda: cache.append(q[:, :2], q[:, :2].half(), pos, pos),
        lambda: cache.append(q[:, :2], q[:, :2], pos.long(), pos),
        lambda: cache.read(pos, pos, dtype=torch.float64),
        lambda: cache.attention(q[:, :3], pos),
        lambda: cache.attention(q, pos[:1]),
        lambda: cache.attention(q, pos, window=-1),
        lambda: cache.attention(q, pos, q_start=pos),
        lambda: cache.attention(q[..., :64], pos),
        lambda: cuda.sample_batch(q[0], w),
        lambda: cuda.sample_batch(q[0].t(), w),
        lambda: cuda.sample_batch(q[0], w[:4], top_k=w[:4]),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
