"""GPU: cases at which the serving operators once answered wrongly or could have, against the plain 64-bit
references of test_gpu_serving.py (its tolerances, unless a test derives its own)."""
import time

import numpy as np
import pytest

from test_gpu_serving import DT, HALF_ULP, T, Case, check_rows, gen, ints, randn, ref_rows, ref_values

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- sampling

def masked_rows(g, rows, vocab, allowed, barred):
    """Logits of constrained rows: all but `allowed` tokens are barred, one of the allowed ones stands well above
    the rest, and of every eight neighbours the first is barred unless it is one of the two largest."""
    torch = T()
    x = torch.full((rows, vocab), barred, device="cuda")
    for b in range(rows):
        ids = torch.randperm(vocab, generator=g, device="cuda")
        ids = ids[ids % 8 != 0][:allowed]
        x[b, ids] = randn(g, len(ids)) * 0.3
        first = torch.randperm((vocab + 7) // 8, generator=g, device="cuda")[:2] * 8
        x[b, first] = torch.tensor([2.5, 2.4], device="cuda")[:len(first)]
    return x


@pytest.mark.parametrize("barred", [float("-inf"), float("nan")])
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("vocab", [64, 5000, 32000, 128256, 400000])
def test_sample_masked_rows(cuda, dt, vocab, barred):
    """Rows that allow a few tokens: none of them is lost on the way to a threshold, whichever path takes the
    row (short list, histogram, both cuts; one CTA to a cluster; rows that are read again at every pass)."""
    torch = T()
    g, rng = gen(vocab), np.random.default_rng(vocab)
    rows, allowed = 24, min(vocab // 3, 3000)
    x = masked_rows(g, rows, vocab, allowed, barred).to(getattr(torch, dt))
    k = [[3, 0, 40, 600, 512, 0, 2, 2000][i % 8] for i in range(rows)]
    p = [[1.0, 0.9, 0.9, 1.0, 0.5, 0.99, 1.0, 0.8][i % 8] for i in range(rows)]
    t = [[1.0, 0.3, 3.0][i % 3] for i in range(rows)]
    u = rng.random(rows).astype(np.float32).tolist()
    assert check_rows(cuda, x, u, t, k, p, [0.0] * rows) <= 3


def test_sample_few_tokens(cuda):
    """Four tokens of 32000: all of the kept ones can be drawn."""
    torch = T()
    x = torch.full((64, 32000), -float("inf"), device="cuda")
    x[:, [8, 16, 25, 33]] = torch.tensor([2.0, 1.9, 1.7, 1.7], device="cuda")
    u = [(i + 0.5) / 64 for i in range(64)]
    for k, p in ((3, 1.0), (0, 0.9), (4, 0.9), (600, 0.95)):
        assert check_rows(cuda, x, u, [1.0] * 64, [k] * 64, [p] * 64, [0.0] * 64) == 0


# ---------------------------------------------------------------- attention

def expire(c):
    """One call of the case with device waits that run out after 5 ms: seconds until the host knows."""
    from blocktensor_b200 import native
    torch = T()
    torch.cuda.synchronize()
    native.call("bt_cuda_kv4_inject_stall", 5)
    try:
        t0 = time.time()
        with pytest.raises(native.CudaBackendError) as e:
            c.run()
        took = time.time() - t0
    finally:
        native.call("bt_cuda_kv4_inject_stall", 0)
    assert e.value.code == native.BT_ERR_DEVICE_TIMEOUT
    return took


@pytest.mark.parametrize("dt,hd", [("float32", 64), ("float16", 128), ("bfloat16", 256)])
@pytest.mark.parametrize("lens", [[40], [5000], [900] * 9, [700, 3, 0, 64, 200] * 40])
def test_attention_waits_run_out(cuda, dt, hd, lens):
    """Waits for copies that give up end the kernel at once (a warp waits five times at most, for its unit
    and for the four copies it has in flight: 25 ms), and the next call is right."""
    torch = T()
    c = Case(cuda, 400 + len(lens), dt, hd, 2, 4, lens, [1] * len(lens), 16)
    good = c.check()
    assert expire(c) < 1.0
    assert torch.equal(c.run(), good)


@pytest.mark.parametrize("dt,hd", [("float16", 64), ("bfloat16", 128)])
@pytest.mark.parametrize("lens,counts,window", [([2000], [300], 0), ([900, 40], [900, 40], 0), ([800] * 40, [200] * 40, 300)])
def test_attention_chunk_waits_run_out(cuda, dt, hd, lens, counts, window):
    """The same in the many-row kernel, with parts of a block on several SMs, masked tiles and several blocks
    a CTA: every warp leaves (seven waits of 5 ms at most)."""
    torch = T()
    c = Case(cuda, 500 + len(lens), dt, hd, 2, 8, lens, counts, 64, window, 4 if window else 0)
    good = c.check()
    assert expire(c) < 1.0
    assert torch.equal(c.run(), good)


@pytest.mark.parametrize("dt,hd", [("float16", 64), ("bfloat16", 128)])
@pytest.mark.parametrize("tokens,n_keys", [(40, 131072), (320, 131072), (1, 131072)])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("bits", [12.5, 24.5, 25.5, 28.5])
def test_attention_peak_over_a_long_tail(cuda, dt, hd, tokens, n_keys, first, bits):
    """One key whose value is 0 stands `bits` powers of two above all others, whose values are 1: the tail's
    share of a row is N / (N + 2^bits).  Of a probability 2^-12 of itself may be lost where it is rounded to
    fp16, or 2^-32 of the row's largest (half a unit of fp16's smallest, 2^-24, with the largest at 2^7 or
    more); of the rest 2^-18; and the result's own rounding."""
    torch = T()
    kv, group = 8, 8
    cache = cuda.KV4Cache(1, n_keys, kv, hd)
    pair = np.array([0, 1], np.float16).view(np.uint8)  # scale 0, min 1
    groups = torch.from_numpy(np.tile(pair, hd // 64)).cuda()
    cache.v_rows[..., hd // 2:] = groups                # ones; keys are zeros
    peak = 0 if first else n_keys - tokens
    cache.k_rows[0, :, peak, hd // 2:] = groups
    cache.v_rows[0, :, peak] = 0
    q = torch.ones(tokens, kv * group, hd, dtype=getattr(torch, dt), device="cuda")
    out = cache.attention(q, ints([n_keys]), q_start=ints([0, tokens]), max_q=tokens, scale=bits * np.log(2.0) / hd)
    cache.check()
    tail = torch.arange(n_keys - tokens, n_keys, device="cuda").double()  # keys that a row sees beside the peak
    want = (tail / (tail + 2.0 ** bits))[:, None, None]
    tol = tail[:, None, None] * 2.0 ** -32 + (2.0 ** -12 + HALF_ULP[dt]) * want + 2.0 ** -18
    assert float(((out.double() - want).abs() / tol).max()) <= 1


# ---------------------------------------------------------------- streams

def operators(cuda, g):
    """Every operator as f(inputs, stream) -> outputs, on inputs (a list of tensors) of its own, at sizes that the
    caching allocator keeps in blocks of their own."""
    torch = T()
    n, kv, hd = 512, 8, 128
    cache = cuda.KV4Cache(n, 64, kv, hd)
    table, w = cuda.rope_table(64, hd), torch.ones(hd, device="cuda")
    slots = torch.arange(n, device="cuda").int()
    pos = torch.arange(n, device="cuda").int() % 64
    lens, u = pos + 1, torch.rand(64, generator=g, device="cuda")
    x = lambda h: randn(g, n, h, hd)  # noqa: E731
    cache.append(x(kv), x(kv), slots, torch.zeros_like(pos))
    return {
        "norms": ([x(16), x(kv)], lambda i, s: cuda.qk_norm_rope(i[0], i[1], w, w, pos, table, stream=s)),
        "append": ([x(16), x(kv), x(kv)],
                   lambda i, s: (cache.append_normed(i[0], i[1], i[2], w, w, slots, pos, table, stream=s),)),
        "read": ([pos.clone()], lambda i, s: cache.read(slots, i[0], torch.float32, stream=s)),
        "attention": ([x(16)], lambda i, s: (cache.attention(i[0], lens, stream=s),)),
        "sample": ([randn(g, 64, 65536)], lambda i, s: cuda.sample_batch(i[0], u, stream=s)),
    }


@pytest.mark.parametrize("name", ["norms", "append", "read", "attention", "sample"])
def test_streams_and_freed_memory(cuda, name):
    """Outputs do not take memory that the current stream still has work on; inputs that the caller drops after
    the call are not reused while it runs; outputs that the caller drops are not while the current stream reads."""
    torch = T()
    inputs, f = operators(cuda, gen(81))[name]
    want = [t.clone() for t in f(inputs, None)]
    side, here = torch.cuda.Stream(), torch.cuda.current_stream()
    torch.cuda.synchronize()
    f(inputs, side)
    torch.cuda.synchronize()

    # freed on the current stream, with a read of it pending there
    old = [torch.full_like(t, 3) for t in want]
    places = {t.data_ptr() for t in old}
    torch.cuda._sleep(100_000_000)
    kept = [t.clone() for t in old]
    del old
    out = f(inputs, side)
    assert not places & {t.data_ptr() for t in out}
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    torch.cuda.synchronize()
    assert all(bool((t == 3).all()) for t in kept)

    # inputs that are dropped while the call has not begun
    mine = [t.clone() for t in inputs]
    places = {t.data_ptr() for t in mine}
    side.wait_stream(here)
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
    out = f(mine, side)
    del mine
    again = [torch.zeros_like(t) for t in inputs]
    assert not places & {t.data_ptr() for t in again}
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))

    # outputs that are dropped while the current stream has not read them
    places = {t.data_ptr() for t in out}
    here.wait_stream(side)
    torch.cuda._sleep(100_000_000)
    kept = [t.clone() for t in out]
    del out
    with torch.cuda.stream(side):
        again = [torch.zeros_like(t) for t in want]
    assert not places & {t.data_ptr() for t in again}
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, want))


# ---------------------------------------------------------------- graphs

def capture(c, lens, out, starts):
    """A graph of two calls, made as a program would that has not called before: no stream given, no call first."""
    torch = T()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for o in out:
            c.cache.attention(c.q, lens, q_start=starts, max_q=max(c.counts), out=o)
    return graph


@pytest.mark.parametrize("lens,counts", [([3000, 300], [1, 1]), ([1500], [200])])
def test_attention_graphs_are_independent(cuda, lens, counts):
    """Graphs captured on one stream, without a call before: the later one replayed first, whatever their
    scratch held; eager calls on the capture stream between them; both at a time on two streams."""
    from blocktensor_b200 import serving
    torch = T()
    c = Case(cuda, 600 + len(lens), "float16", 128, 2, 8, lens, counts, 64)
    starts = None if max(counts) == 1 else c.starts
    want = c.check()
    at = ints(lens)
    outs = [[torch.zeros_like(c.q) for _ in range(2)] for _ in range(2)]
    torch.cuda.synchronize()
    known = set(serving._workspaces)
    graphs = [capture(c, at, o, starts) for o in outs]
    assert set(serving._workspaces) == known  # nothing of a capture serves eager calls
    for kept in (serving._workspaces, serving._captured):
        for key, ws in kept.items():
            if key not in known:
                ws[2].fill_(255)
    for g in (1, 0):
        graphs[g].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs[g])
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    with torch.cuda.stream(torch.cuda.graph.default_capture_stream):
        eager = c.cache.attention(c.q, at, q_start=starts, max_q=max(counts))
    torch.cuda.synchronize()
    assert torch.equal(eager, want)
    for _ in range(20):
        for g in range(2):
            for o in outs[g]:
                o.zero_()
        for g in range(2):
            side[g].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side[g]):
                for _ in range(10):
                    graphs[g].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for g in range(2) for o in outs[g])
    c.cache.check()


def test_attention_graph_with_branches(cuda):
    """Calls on two streams of one capture do not share scratch."""
    torch = T()
    c = Case(cuda, 620, "bfloat16", 64, 2, 4, [5000], [1], 16)
    want, at = c.check(), ints([5000])
    outs = [torch.zeros_like(c.q) for _ in range(8)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        for i, o in enumerate(outs):
            c.cache.attention(c.q, at, out=o, stream=side if i % 2 else None)
        here.wait_stream(side)
    for _ in range(20):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("counts", [[1], [200]])
def test_attention_after_a_timeout(cuda, counts):
    """Whatever an expired wait left in the scratch, the next call begins with cleared tickets."""
    from blocktensor_b200 import native, serving
    torch = T()
    c = Case(cuda, 630, "float16", 64, 2, 4, [3000], counts, 16)
    good = c.check()
    for ws in serving._workspaces.values():
        ws[2].fill_(255)
    c.cache.status.fill_(native.BT_KV4_TIMEOUT)
    with pytest.raises(native.CudaBackendError):
        c.cache.check()
    assert torch.equal(c.run(), good)


@pytest.mark.parametrize("vocab", [100, 60000, 400000])
def test_sample_nan_parameters(cuda, vocab):
    """A NaN temperature is greedy, a NaN top-p or min-p cuts nothing, and a NaN u draws as 0 does."""
    torch = T()
    g, rows = gen(vocab), 8
    x = randn(g, rows, vocab)
    x[1::2, vocab // 2:vocab // 2 + 5] = 9.0  # equal maxima
    f = lambda v: torch.full((rows,), v, device="cuda")  # noqa: E731
    u, nan = torch.linspace(0, 0.99, rows, device="cuda"), f(float("nan"))
    for k in (None, torch.full((rows,), 40, dtype=torch.int32, device="cuda")):
        same = lambda a, b: all(torch.equal(s, t) for s, t in zip(a, b))  # noqa: E731
        assert same(cuda.sample_batch(x, u, nan, k), cuda.sample_batch(x, u, f(0.0), k))
        assert same(cuda.sample_batch(x, u, None, k, nan, None), cuda.sample_batch(x, u, None, k))
        assert same(cuda.sample_batch(x, u, None, k, None, nan), cuda.sample_batch(x, u, None, k))
        assert same(cuda.sample_batch(x, nan, None, k), cuda.sample_batch(x, f(0.0), None, k))


@pytest.mark.parametrize("dt,hd", [("float32", 64), ("bfloat16", 64), ("bfloat16", 128), ("bfloat16", 256), ("float32", 256)])
@pytest.mark.parametrize("lens,counts", [([1], [1]), ([300, 2, 1], [1, 1, 1]), ([40], [40]), ([700], [120])])
@pytest.mark.parametrize("size", [1e25, 1e31, 1e35, 1e36])
def test_attention_huge_queries(cuda, dt, hd, lens, counts, size):
    """Queries so large that one key takes all: scores of either sign up to what fp32 holds.  Rows whose best two
    scores lie within 2 % of the largest are not judged (the order of such may turn with fp16 operands)."""
    torch = T()
    c = Case(cuda, 640, dt, hd, 2, 4, lens, counts)
    c.q.copy_((c.q.float() * (size / 10)).to(c.q.dtype))
    got, (want, _) = c.run().double(), c.want()
    row = judged = 0
    for i, (length, count) in enumerate(zip(lens, counts)):
        q_at = torch.arange(length - count, length, device="cuda")
        for h in range(8):
            k, v = c.k[i][:, h // 4], c.v[i][:, h // 4]
            s = (c.q[row:row + count, h].double() @ k.T).masked_fill(torch.arange(length, device="cuda") > q_at[:, None], -np.inf)
            best = s.topk(min(2, length), -1).values
            second = best[:, 1] if length > 1 else torch.full_like(best[:, 0], -np.inf)
            clear = best[:, 0] - second > 0.02 * s.masked_fill(s == -np.inf, 0).abs().amax(-1)
            tol = (2.0 ** -18 if dt == "float32" else 2.0 ** -11) * v.abs().max() + HALF_ULP[dt] * want[row:row + count, h].abs()
            err = (got[row:row + count, h] - want[row:row + count, h]).abs()
            assert bool((err <= tol)[clear].all())
            judged += int(clear.sum())
        row += count
    assert judged >= 4 * sum(counts) and bool(got.isfinite().all())


# ---------------------------------------------------------------- attention, every key counted

ROUND = {"float16": 2.0 ** -12, "bfloat16": 2.0 ** -9}  # rms of the result's own rounding, relative


def deviations(c, got):
    """The errors of 16-bit attention in standard deviations of what its roundings add up to: keys, values and
    probabilities held to 2^-12 rms each (a key moves a score by 2^-12 sqrt(sum (q k)^2), and that score's share
    of the result by p (v - o)), independent of one another, and the result's rounding.  A key left out or
    counted twice among n alike moves a row by |v - o| / n, some 2^11 / sqrt(n) of these."""
    torch = T()
    out, row = [], 0
    for i, (length, count) in enumerate(zip(c.lens, c.counts)):
        if length == 0 or count == 0:
            assert bool((got[row:row + count] == 0).all())
            row += count
            continue
        at, q_at = torch.arange(length, device="cuda"), torch.arange(length - count, length, device="cuda")[:, None]
        seen = at <= q_at
        if c.window:
            seen &= (at > q_at - c.window) | (at < c.sinks)
        for h in range(c.kv * c.group):
            k, v = c.k[i][:, h // c.group], c.v[i][:, h // c.group]
            q = c.q[row:row + count, h].double() * c.scale
            p = torch.nan_to_num(torch.softmax((q @ k.T).masked_fill(~seen, -np.inf), -1))
            o = p @ v
            p2 = p.pow(2)
            w = p2 * (q.pow(2) @ k.pow(2).T)
            var = 2 * p2 @ v.pow(2) + w @ v.pow(2) - 2 * o * (w @ v) + o.pow(2) * w.sum(-1, keepdim=True)
            dev = (2.0 ** -24 * var + (ROUND[c.dt] * o).pow(2) + 2.0 ** -46 * v.abs().max() ** 2).sqrt()
            out.append((got[row:row + count, h].double() - o) / dev)
        row += count
    return torch.cat([x.flatten() for x in out])


def check_rms(c, **kw):
    """Within 1.25 of these deviations (upper bounds) in the root mean square over thousands of elements."""
    d = float(deviations(c, c.run(**kw)).pow(2).mean().sqrt())
    assert d <= 1.25, d


CALLS = [
    # lens, counts, kv, group, page, window, sinks
    ([700, 33, 129, 64, 255], [1] * 5, 2, 4, 64, 0, 0),
    ([4097], [1], 2, 8, 16, 0, 0),
    ([900, 3, 400, 40, 0], [1] * 5, 2, 8, 16, 100, 4),
    ([1023, 1025, 65, 63, 1], [1] * 5, 4, 1, 16, 0, 0),
    ([700], [100], 1, 8, 0, 0, 0),
    ([129, 700, 128, 31], [128, 200, 127, 31], 2, 3, 32, 0, 0),
    ([2049], [130], 2, 4, 16, 0, 0),
    ([1100], [600], 4, 8, 256, 400, 1),
    ([260, 20, 400], [260, 20, 5], 2, 8, 16, 33, 70),
]


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("i", range(len(CALLS)))
def test_attention_rms(cuda, dt, hd, i):
    lens, counts, kv, group, page, window, sinks = CALLS[i]
    check_rms(Case(cuda, 700 + i, dt, hd, kv, group, lens, counts, page, window, sinks, shuffle=i % 2 == 0))


def count_keys(cuda, seed, dt, hd, kv, group, lens, counts, page=0, window=0, sinks=0, flagged=None):
    """Queries of zeros give every key that a row sees the same weight, and key j's value is 1 in element j % hd
    and 0 elsewhere (zeros too unless j is in `flagged`): times their number, a row of the result counts the keys.
    Probabilities, their sums and the products are powers of two and small whole numbers, so that what is left is
    the result's rounding and an fp32 reciprocal's.  What no row sees is NaN, pages of it are not in the table."""
    torch = T()
    g, n, max_seq = gen(seed), len(lens), max(lens) + 3
    cache = cuda.KV4Cache(n, max_seq, kv, hd, page_tokens=page, n_pages=n * -(-max_seq // page) if page else 0)
    if page:
        cache.page_table[:] = torch.randperm(cache.n_pages, generator=g, device="cuda").int().view(n, -1)
    k = torch.randint(0, 256, (kv, hd // 2 + hd // 16), generator=g, device="cuda", dtype=torch.uint8)
    k[:, hd // 2:] = torch.tensor([0.3, -2.0], device="cuda").half().view(torch.uint8).repeat(hd // 64)
    cache.k_rows.fill_(0xFF)
    cache.v_rows.fill_(0xFF)
    one = torch.tensor([1.0, 0.0], device="cuda").half().view(torch.uint8).repeat(hd // 64)
    want = []
    for i, (length, count) in enumerate(zip(lens, counts)):
        at, q_at = torch.arange(length, device="cuda"), torch.arange(length - count, length, device="cuda")[:, None]
        seen = at <= q_at
        if window:
            seen &= (at > q_at - window) | (at < sinks)
        live = at[seen.any(0)]
        rows = torch.zeros(length, hd // 2 + hd // 16, dtype=torch.uint8, device="cuda")
        flag = torch.ones_like(at, dtype=torch.bool) if flagged is None else (at >= flagged[0]) & (at < flagged[1])
        rows[at, at % hd // 2] = torch.where(flag, 1 << 4 * (at % 2), 0).to(torch.uint8)
        rows[:, hd // 2:] = one
        p = cache.page_table[i, live // page].long() if page else torch.full_like(live, i)
        cache.v_rows[p, :, live % cache.page_tokens] = rows[live][:, None]
        cache.k_rows[p, :, live % cache.page_tokens] = k
        if page:
            gone = torch.ones(cache.max_pages, dtype=torch.bool, device="cuda")
            gone[live // page] = False
            cache.page_table[i][gone] = -1
        onehot = torch.zeros(length, hd, dtype=torch.float64, device="cuda")
        onehot[at, at % hd] = flag.double()
        want.append(seen.double() @ onehot / seen.sum(1, keepdim=True).clamp(min=1))
    q = torch.zeros(sum(counts), kv * group, hd, dtype=getattr(torch, dt), device="cuda")
    starts = None if all(c == 1 for c in counts) else ints(np.concatenate([[0], np.cumsum(counts)]).tolist())
    out = cache.attention(q, ints(lens), q_start=starts, max_q=max(counts), window=window, sinks=sinks)
    cache.check()
    want = torch.cat(want)[:, None]
    assert bool(((out.double() - want).abs() <= (HALF_ULP[dt] + 2.0 ** -22) * want).all())


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("i", range(len(CALLS)))
def test_attention_counts_every_key(cuda, dt, hd, i):
    lens, counts, kv, group, page, window, sinks = CALLS[i]
    count_keys(cuda, 750 + i, dt, hd, kv, group, lens, counts, page, window, sinks)


@pytest.mark.parametrize("dt,hd,group,count", [("float16", 64, 8, 1), ("float32", 128, 4, 1), ("float16", 128, 8, 20),
                                               ("bfloat16", 64, 8, 130)])
def test_attention_counts_every_key_of_many(cuda, dt, hd, group, count):
    """100003 keys, 32 an element at a time."""
    for lo in range(0, 100003, 32 * hd):
        count_keys(cuda, 770, dt, hd, 1, group, [100003], [count], flagged=(lo, lo + 32 * hd))


@pytest.mark.parametrize("dt,hd", [("float16", 64), ("bfloat16", 128)])
@pytest.mark.parametrize("n", [33, 64, 65, 150])
def test_attention_many_prompts(cuda, dt, hd, n):
    """More sequences with many rows than a warp has lanes and than the kernel keeps at hand, short ones and
    empty ones among them."""
    lens = [[90, 1, 40, 0, 130, 7][i % 6] + i % 5 for i in range(n)]
    counts = [[40, 1, 33, 0, 130, 7][i % 6] for i in range(n)]
    check_rms(Case(cuda, 720 + n, dt, hd, 2, 4, lens, counts, 16, shuffle=True))
    count_keys(cuda, 720 + n, dt, hd, 2, 4, lens, counts, 16)


@pytest.mark.parametrize("dt,hd", [("float32", 64), ("float16", 128), ("bfloat16", 256)])
@pytest.mark.parametrize("n", [257, 513, 1100])
def test_attention_many_sequences(cuda, dt, hd, n):
    """More sequences than a CTA of the few-row kernel has threads."""
    lens = [[1, 17, 40, 0, 33][i % 5] for i in range(n - 1)] + [300]
    Case(cuda, 730 + n, dt, hd, 2, 4, lens, [1] * n, 16).check()
    count_keys(cuda, 730 + n, dt, hd, 2, 4, lens, [1] * n, 16)


def test_attention_chunk_past_4gb(cuda):
    """The many-row kernel on rows beyond the first 4 GB of the pool."""
    torch = T()
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    g, kv, group, hd, max_seq = gen(62), 4, 4, 128, 2_200_000  # 72 B * 4 * 2.2 M = 0.63 GB a slot, 8 slots a side
    cache = cuda.KV4Cache(8, max_seq, kv, hd)
    length, window, count = 2_100_000, 300, 100
    first = length - count + 1 - window
    pos = torch.arange(first, length, device="cuda").int()
    for lo in range(0, len(pos), 128):
        p = pos[lo:lo + 128]
        cache.append(randn(g, len(p), kv, hd), randn(g, len(p), kv, hd), torch.full_like(p, 7), p)
    q = randn(g, count, kv * group, hd).half()
    out = cache.attention(q, ints([length]), q_start=ints([0, count]), slots=ints([7]), max_q=count, window=window)
    cache.check()
    # the same rows at the start of a small cache, with the window's edge as it lies
    small = cuda.KV4Cache(1, len(pos), kv, hd)
    small.k_rows[0, :, :len(pos)] = cache.k_rows[7, :, first:length]
    small.v_rows[0, :, :len(pos)] = cache.v_rows[7, :, first:length]
    kk, vv = (ref_values(r[0, :, :len(pos)], hd) for r in (small.k_rows, small.v_rows))
    at, q_at = torch.arange(first, length, device="cuda"), torch.arange(length - count, length, device="cuda")[:, None]
    seen = (at <= q_at) & (at > q_at - window)
    for h in range(kv * group):
        k, v = kk[h // group], vv[h // group]
        p = torch.softmax((q[:, h].double() @ k.T * hd ** -0.5).masked_fill(~seen, -np.inf), -1)
        # (the tolerance of test_attention_past_4gb, which these sizes keep to alike)
        assert float((out[:, h].double() - p @ v).abs().max()) <= (6 * 1.0 + 4) * 2.0 ** -11 * float(v.abs().max())


@pytest.mark.parametrize("dt,hd", [("float16", 64), ("bfloat16", 128)])
def test_attention_rows_of_no_sequence(cuda, dt, hd):
    """Rows of q before the first sequence's, between none and after the last one's are not written."""
    torch = T()
    c = Case(cuda, 740, dt, hd, 2, 4, [50, 300], [1, 60])
    want = c.run(out=torch.full_like(c.q, 5))
    pad = torch.zeros(7, *c.q.shape[1:], dtype=c.q.dtype, device="cuda")
    q = torch.cat([pad[:3], c.q, pad])
    out = torch.full_like(q, 5)
    c.cache.attention(q, ints(c.lens), q_start=c.starts + 3, max_q=60, out=out)
    c.cache.check()
    assert torch.equal(out[3:-7], want) and bool((out[:3] == 5).all()) and bool((out[-7:] == 5).all())


# ---------------------------------------------------------------- cached keys, as bt_cuda.h defines them

def defined_key(x, w, eps, cos, sin):
    """The norm and rotation of bt_cuda_kv4_append in numpy fp32, operation by operation (rsqrtf by the device)."""
    torch = T()
    s = x * x
    hd = x.shape[-1]
    if hd == 256:
        s = s[..., :128] + s[..., 128:]
    if hd == 64:
        s = s[..., :32] + s[..., 32:]
    else:
        four = s.reshape(*s.shape[:-1], 32, 4)
        s = ((four[..., 0] + four[..., 1]) + four[..., 2]) + four[..., 3]
    while s.shape[-1] > 1:
        half = s.shape[-1] // 2
        s = s[..., :half] + s[..., half:]
    mean = s * np.float32(1 / hd) + np.float32(eps)
    x = x * torch.rsqrt(torch.from_numpy(mean).cuda()).cpu().numpy() * w
    h = cos.shape[-1]
    a, b = x[..., :h], x[..., h:2 * h]
    return np.concatenate([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]], -1)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("hd,rot", [(64, 64), (64, 16), (128, 128), (128, 96), (256, 256), (256, 64)])
def test_append_codes_as_defined(cuda, dt, hd, rot):
    torch = T()
    g, tokens, kv = gen(hd + rot), 700, 3
    k, v = ((randn(g, tokens, kv, hd) * (1 + 2 * torch.rand(hd, generator=g, device="cuda"))).to(getattr(torch, dt)) for _ in range(2))
    w, table = 1 + 0.3 * randn(g, hd), cuda.rope_table(tokens, rot, 500000.0)
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda")
    cache = cuda.KV4Cache(1, tokens, kv, hd)
    cache.append_normed(torch.zeros_like(k), k, v, None, w, torch.zeros_like(pos), pos, table, 1e-5)
    cos, sin = (table[:, None, :, i].cpu().numpy() for i in (0, 1))
    want = defined_key(k.float().cpu().numpy(), w.cpu().numpy(), 1e-5, cos, sin)
    assert want.dtype == np.float32
    assert np.array_equal(cache.k_rows[0, :, :tokens].transpose(0, 1).cpu().numpy(), ref_rows(torch.from_numpy(want)))


# ---------------------------------------------------------------- the decoder

def test_decoder_refusals(cuda):
    """A slot named twice, a slot without tokens, tokens that do not add up: refused before anything is kept."""
    from blocktensor_b200.serve4 import Decoder4, Shape
    torch = T()
    m = Decoder4(Shape(vocab=256, dim=128, hidden=256, layers=1, heads=2, kv_heads=1, head_dim=64), 2, 64, page_tokens=16)
    free, u = m.caches[0].pages(), torch.full((2,), 0.5, device="cuda")
    for prompts, slots in (([[1, 2], []], [0, 1]), ([[1], [2]], [0, 0]), ([], []), ([[1]], [0, 1])):
        with pytest.raises(ValueError):
            m.prefill(prompts, slots, u)
    with pytest.raises(ValueError):
        m.forward(torch.ones(3, dtype=torch.int64, device="cuda"), [0, 1], [1, 1])
    assert m.caches[0].pages() == free and m.lens == [0, 0]
    assert m.prefill([[1, 2], [3]], [0, 1], u).shape == (2,)
    m.check()


def test_attention_integer_refusals(cuda):
    """Numbers past 32 bits are refused as other arguments are."""
    torch = T()
    c, q = cuda.KV4Cache(1, 16, 1, 64), torch.zeros(1, 1, 64, device="cuda")
    for kw in (dict(window=1 << 32), dict(window=9, sinks=1 << 32), dict(max_q=1 << 32), dict(sinks=-1), dict(scale=float("nan")),
               dict(scale=1e39)):
        with pytest.raises(ValueError):
            c.attention(q, ints([1]), **kw)


@pytest.mark.parametrize("dt,hd", [("float32", 64), ("float16", 128), ("bfloat16", 64), ("bfloat16", 256)])
@pytest.mark.parametrize("counts", [[1, 1], [90, 40]])
def test_attention_nan_and_infinite_queries(cuda, dt, hd, counts):
    """A NaN or infinite element makes its own (query, head) row NaN and no other one."""
    torch = T()
    c = Case(cuda, 760, dt, hd, 2, 4, [500, 77], counts, 16)
    want = c.check()
    bad = [(0, 0, float("nan")), (sum(counts) // 2, 3, float("inf")), (sum(counts) - 1, 7, -float("inf"))]
    for row, head, v in bad:
        c.q[row, head, 5] = v
    got = c.run()
    for row, head, _ in bad:
        assert bool(got[row, head].isnan().all())
        got[row, head] = want[row, head]
    assert torch.equal(got, want)


def test_check_waits_for_every_stream(cuda):
    """check() sees what a call on another stream, not yet begun, will report."""
    torch = T()
    c, x = cuda.KV4Cache(2, 40, 1, 64), torch.ones(1, 1, 64, device="cuda")
    slots, pos, side = ints([5]), ints([0]), torch.cuda.Stream()
    c.append(x, x, pos, pos, stream=side)  # (a kernel's first launch waits for the device)
    c.check()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
    c.append(x, x, slots, pos, stream=side)
    with pytest.raises(IndexError):
        c.check()
    c.check()


def test_broadcast_outputs_are_refused(cuda):
    """An output whose rows share memory would be written by several threads at a time."""
    torch = T()
    q, w, pos, table = torch.zeros(2, 4, 128, device="cuda"), torch.ones(128, device="cuda"), ints([0, 1]), cuda.rope_table(4, 128)
    c = cuda.KV4Cache(2, 32, 2, 128)
    for shared in (torch.zeros(1, 4, 128, device="cuda").expand(2, 4, 128), torch.zeros(2, 1, 128, device="cuda").expand(2, 4, 128)):
        with pytest.raises(ValueError):
            cuda.qk_norm_rope(q, None, w, None, pos, table, q_out=shared)
        with pytest.raises(ValueError):
            c.attention(q, pos, out=shared)
        with pytest.raises(ValueError):
            c.append_normed(q, q[:, :2], q[:, 2:], w, w, pos, pos, table, q_out=shared)
        # as an input it is read as any other
        a, _ = cuda.qk_norm_rope(shared, None, w, None, pos, table)
        assert torch.equal(a, torch.zeros_like(q))
    one = torch.zeros(1, 4, 128, device="cuda").as_strided((1, 4, 128), (0, 128, 1))
    cuda.qk_norm_rope(q[:1], None, w, None, pos[:1], table, q_out=one)
