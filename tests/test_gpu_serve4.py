"""GPU: the small decoder on 4-bit caches against a 64-bit forward pass of the same quantised weights
and 4-bit keys and values, at every prompt position and decode step.

Tolerance: the int8 products carry 2^-21 of their inputs, attention and norms 2^-18; what is left is a
4-bit code that falls the other way where its value lies within rounding of a half, a change of one step
(about a third of the row's deviation) in one element of one key, which moves a logit by far less than
1 % of the logits' deviation.
"""
import math

import pytest

pytestmark = pytest.mark.gpu


def held(x):
    """What 4-bit rows of x [..., hd] (float64) stand for."""
    g = x.unflatten(-1, (-1, 64))
    low = g.amin(-1, keepdim=True)
    scale = ((g.amax(-1, keepdim=True) - low) / 15).half().double()
    low = low.half().double()
    return (((g - low) / scale).round().clamp(0, 15) * scale + low).flatten(-2)


class Reference:
    def __init__(self, bt, model):
        import torch
        self.torch, self.m, self.s = torch, model, model.shape
        self.w = lambda mat: bt.dequantize_q8_0(mat.blocks).view(mat.M, mat.K).double()

    def norm(self, x, w):
        return x / (x.pow(2).mean(-1, keepdim=True) + self.s.eps).sqrt() * w.double()

    def turn(self, x, pos):
        half = self.s.head_dim // 2
        c, s = (self.m.rope[pos].double()[:, None, :, i] for i in (0, 1))
        a, b = x[..., :half], x[..., half:]
        return self.torch.cat([a * c - b * s, b * c + a * s], -1)

    def logits(self, tokens):
        """Of every position of one sequence."""
        torch, s, m = self.torch, self.s, self.m
        n = len(tokens)
        pos = torch.arange(n, device="cuda")
        seen = pos <= pos[:, None]
        if m.window:
            seen &= (pos > pos[:, None] - m.window) | (pos < m.sinks)
        x = m.embed[torch.tensor(tokens, device="cuda")].double()
        for w in m.layers:
            h = (self.norm(x, w["attn_norm"]) @ self.w(w["qkv"]).T).view(n, -1, s.head_dim)
            q, k, v = h.split([s.heads, s.kv_heads, s.kv_heads], 1)
            q = self.turn(self.norm(q, w["q_norm"]), pos)
            k, v = held(self.turn(self.norm(k, w["k_norm"]), pos)), held(v)
            k, v = (t.repeat_interleave(s.heads // s.kv_heads, 1) for t in (k, v))
            p = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(s.head_dim)
            p = p.masked_fill(~seen, -math.inf).softmax(-1)
            x = x + torch.einsum("hij,jhd->ihd", p, v).reshape(n, -1) @ self.w(w["o"]).T
            gate, up = (self.norm(x, w["ffn_norm"]) @ self.w(w["up"]).T).chunk(2, 1)
            x = x + (torch.nn.functional.silu(gate) * up) @ self.w(w["down"]).T
        return self.norm(x, m.out_norm) @ self.w(m.head).T


def close(got, want):
    err = (got.double() - want).abs().max() / want.std()
    assert float(err) <= 0.01, float(err)


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_decoder(cuda, window, sinks):
    import torch
    from blocktensor_b200.serve4 import Decoder4, Shape
    shape = Shape(vocab=1000, dim=256, hidden=512, layers=2, heads=6, kv_heads=2, head_dim=64)
    m = Decoder4(shape, 3, 256, page_tokens=16, n_pages=12, window=window, sinks=sinks, seed=5)
    ref = Reference(cuda, m)
    g = torch.Generator("cuda").manual_seed(9)
    prompts = [torch.randint(0, 1000, (n,), generator=g, device="cuda").tolist() for n in (1, 57, 20)]
    slots = [2, 0, 1]
    # prompts of uneven lengths together
    logits = m.forward(torch.tensor([t for p in prompts for t in p], device="cuda"), slots, [len(p) for p in prompts])
    row = 0
    for p in prompts:
        close(logits[row:row + len(p)], ref.logits(p))
        row += len(p)
    # then single tokens, greedy and drawn, and a chunk of one sequence beside a token of another
    history = [list(p) for p in prompts]
    m.next[slots] = torch.tensor([3, 7, 11], dtype=torch.int32, device="cuda")
    for i, t in enumerate((3, 7, 11)):
        history[i].append(t)
    for _ in range(3):
        logits = m.forward(m.next[slots], slots, [1, 1, 1])
        for i in range(3):
            close(logits[i:i + 1], ref.logits(history[i])[-1:])
        token = m._draw(logits, slots, torch.tensor([0.2, 0.5, 0.9], device="cuda"),
                        dict(temperature=torch.tensor([0.0, 1.0, 0.7], device="cuda")))
        assert int(token[0]) == int(logits[0].argmax())
        for i, t in enumerate(token.tolist()):
            history[i].append(t)
    more = torch.randint(0, 1000, (9,), generator=g, device="cuda").tolist()
    logits = m.forward(torch.tensor(history[0][-1:] + more, device="cuda"), [2, 0], [1, 9])
    close(logits[:1], ref.logits(history[0])[-1:])
    close(logits[1:], ref.logits(history[1][:-1] + more)[-9:])
    m.check()
    # a slot's pages go back and serve another sequence
    free = m.caches[0].pages()[0]
    m.release(0)
    assert m.caches[0].pages()[0] > free
    close(m.forward(torch.tensor(prompts[2], device="cuda"), [0], [20]), ref.logits(prompts[2]))
    with pytest.raises(MemoryError):
        m.forward(torch.zeros(230, dtype=torch.int64, device="cuda"), [0], [230])


def test_command(cuda, capsys):
    from blocktensor_b200 import serve4
    serve4.main(["--steps", "3", "--slots", "2", "--window", "32", "--sinks", "2"])
    first = capsys.readouterr().out
    serve4.main(["--steps", "3", "--slots", "2", "--window", "32", "--sinks", "2"])
    assert first == capsys.readouterr().out and first.count("slot") == 2
