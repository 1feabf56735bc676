"""GPU: cases at which the serving operators once answered wrongly or could have, against the plain 64-bit
references of test_gpu_serving.py (its tolerances, unless a test derives its own)."""
import time

import numpy as np
import pytest

from test_gpu_serving import DT, HALF_ULP, T, Case, check_rows, gen, ints, randn

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
