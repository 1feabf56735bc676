"""Serving operators on torch CUDA tensors: head norms with rotation, 4-bit K/V caches with the
attention over them, batched sampling (bt_cuda_qk_norm_rope, bt_cuda_kv4_*, bt_cuda_sample_batch in
include/bt_cuda.h, which states their mathematics).

Activations are fp32, fp16 or bf16 tensors whose last dimension is contiguous; every call checks its
arguments (ValueError), launches on torch's current stream or on ``stream``, and does not synchronise.
With ``stream`` the call is as if made under ``torch.cuda.stream(stream)``: the caller orders the two
streams; what the call allocates is that stream's, and no tensor that it was given or returns is reused
before both streams are done with it.
Index tensors (positions, slots, lengths) are int32 on the device; values out of range are never
followed and show in :meth:`KV4Cache.check`.
"""
from __future__ import annotations

import ctypes as C
from struct import Struct

import torch

from . import native
from .native import BT_BF16, BT_F16, BT_F32, KV4, KV4AttnArgs, QkArgs, SampleArgs

__all__ = ["KV4Cache", "qk_norm_rope", "rope_table", "sample_batch"]

_DTYPES = {torch.float32: BT_F32, torch.float16: BT_F16, torch.bfloat16: BT_BF16}
_NO_HEADS = (0, 0, 0)

# The argument structs packed in one step: a call on one token is bound by the host, and a
# ctypes structure takes several microseconds to fill.
_pack_qk = Struct("<" + "Qqq" * 5 + "5Q6Iif")
_pack_attn = Struct("<" + "Qqq" * 2 + "3Q6Iif")
_pack_sample = Struct("<Qq7Q2IiI")
assert (_pack_qk.size, _pack_attn.size, _pack_sample.size) == (C.sizeof(QkArgs), C.sizeof(KV4AttnArgs), C.sizeof(SampleArgs))

_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice

# (device, stream) -> (pointer, bytes, tensor): the attention's scratch, kept as calls of one
# stream follow one another.  Calls that are captured take one of their capture's own (the
# fourth member is its number), which the graph clears at every replay: graphs may be replayed
# in any order and beside one another and calls.
_workspaces = {}
_captured = {}
_is_capturing = torch._C._cuda_isCurrentStreamCapturing


def _new_workspace(cache, dev, s, capture):
    with torch.cuda.device(dev):
        size = native.load().bt_cuda_kv4_attention_workspace()
        mem = torch.empty(size, dtype=torch.uint8, device="cuda")
        mem[:native.BT_KV4_WORKSPACE_ZERO].zero_()
    ws = cache[dev, s] = (mem.data_ptr(), size, mem, capture)
    return ws


def _dtype(t) -> int:
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise ValueError(f"expected a float32, float16 or bfloat16 tensor, got {t.dtype}")
    return d


def _heads(t, name, shape=None, dtype=None, dev=None):
    """(pointer, token stride, head stride) of a [tokens, heads, head_dim] tensor (of the given shape, type
    and device)."""
    strides = t.stride()
    if len(strides) != 3 or not t.is_cuda:
        raise ValueError(f"{name}: expected a [tokens, heads, head_dim] CUDA tensor")
    if strides[2] != 1 and t.shape[2] > 1:
        raise ValueError(f"{name}: the elements of a head must be contiguous")
    if shape is not None and (t.shape != shape or t.dtype is not dtype or t.get_device() != dev):
        raise ValueError(f"{name}: tokens, heads, head_dim, dtype or device do not match")
    return t.data_ptr(), strides[0], strides[1]


def _out(t, name, shape, like, dev):
    """(tensor, (pointer, strides)): the caller's output, checked, or a new one."""
    if t is None:
        # (empty_like keeps strides, so it only serves contiguous tensors; 0.5 us less than new_empty)
        t = torch.empty_like(like) if like.is_contiguous() else like.new_empty(shape)
        return t, (t.data_ptr(), shape[1] * shape[2], shape[2])
    h = _heads(t, name, shape, like.dtype, dev)
    if (h[1] == 0 and shape[0] > 1) or (h[2] == 0 and shape[1] > 1):
        raise ValueError(f"{name}: rows of an output must not share memory")
    return t, h


def _vector(t, name, n, dtype, dev):
    if t.dtype is not dtype or t.numel() != n or not t.is_contiguous() or t.get_device() != dev:
        raise ValueError(f"{name}: expected {n} contiguous {dtype} values on cuda:{dev}")
    return t.data_ptr()


def _elsewhere(stream):
    """Whether a call has to change streams."""
    return stream.cuda_stream != _raw_stream(stream.device_index)


def _on_stream(stream, keep, f, *args):
    """f(*args) on ``stream``; ``keep``: tensors that it uses beside its arguments."""
    here = torch.cuda.current_stream(stream.device)
    given = [t for t in (*args, *keep) if isinstance(t, torch.Tensor) and t.is_cuda]
    if any(t.get_device() != stream.device_index for t in given):
        raise ValueError("stream: of another device than the tensors")
    with torch.cuda.stream(stream):
        out = f(*args)
    for t in given:
        t.record_stream(stream)
    for t in out if isinstance(out, tuple) else (out,):
        if t is not None and not any(t is g for g in given):
            t.record_stream(here)
    return out


def _launch(fn, name, dev, *args):
    """The C call on the tensors' device and its current stream."""
    s = _raw_stream(dev)
    if dev == _current_device():
        rc = fn(*args, s)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, s)
    if rc:
        native.check(rc, name)


def rope_table(positions: int, rot_dim: int, theta: float = 10000.0, device="cuda"):
    """cos and sin of cpu_ref::rope's angles (cpu_ref.hpp:38-41) for positions 0 .. positions - 1, taken
    in double precision: [positions, rot_dim / 2, 2] fp32."""
    if rot_dim <= 0 or rot_dim % 16:
        raise ValueError("rope_table: rot_dim must be a positive multiple of 16")
    freq = theta ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], -1).float().to(device)


def _rope(table, dev):
    if table is None:
        return 0, 0, 0
    if table.dim() != 3 or table.dtype is not torch.float32 or not table.is_contiguous() or table.get_device() != dev:
        raise ValueError("table: expected a contiguous [positions, rot_dim / 2, 2] float32 tensor on the queries' device")
    n, half, two = table.shape
    if two != 2:
        raise ValueError("table: expected (cos, sin) pairs in its last dimension")
    return table.data_ptr(), n, 2 * half


def qk_norm_rope(q, k, q_weight, k_weight, positions, table, eps: float = 1e-5, q_out=None, k_out=None, stream=None):
    """Norms of each head of q [T, H, hd] and k [T, KVH, hd] and their rotation, one pass over both
    (bt_cuda_qk_norm_rope).  q_weight / k_weight: [hd] float32, or None for no norm; table: rope_table(),
    or None for no rotation; positions: [T] int32.  q_out / k_out may be q and k.  k may be None."""
    if stream is not None and _elsewhere(stream):
        return _on_stream(stream, (), qk_norm_rope, q, k, q_weight, k_weight, positions, table, eps, q_out, k_out)
    qh = _heads(q, "q")
    shape, dtype, dev = q.shape, q.dtype, q.get_device()
    tokens, heads, hd = shape
    q_out, qoh = _out(q_out, "q_out", shape, q, dev)
    kh = koh = _NO_HEADS
    kv_heads = 0
    if k is not None:
        kv_heads = k.shape[1] if k.dim() == 3 else 0
        k_shape = (tokens, kv_heads, hd)
        kh = _heads(k, "k", k_shape, dtype, dev)
        k_out, koh = _out(k_out, "k_out", k_shape, k, dev)
    a = _pack_qk.pack(*qh, *kh, *_NO_HEADS, *qoh, *koh,
                      0 if q_weight is None else _vector(q_weight, "q_weight", hd, torch.float32, dev),
                      0 if k_weight is None else _vector(k_weight, "k_weight", hd, torch.float32, dev),
                      _vector(positions, "positions", tokens, torch.int32, dev), 0,
                      *_rope(table, dev), tokens, heads, kv_heads, hd, _dtype(q), eps)
    _launch(native.load().bt_cuda_qk_norm_rope, "bt_cuda_qk_norm_rope", dev, a)
    return q_out, k_out


class KV4Cache:
    """A 4-bit cache of one layer (bt_kv4): ``n_seq`` slots of up to ``max_seq`` positions.

    Contiguous by default.  With ``page_tokens`` the rows live in a pool of ``n_pages`` pages;
    :meth:`reserve` and :meth:`release` hand them out (of several layers, the first one's ``page_table``
    given to the others serves all), or a ``page_table`` the caller keeps is read as it is.  ``k_rows`` /
    ``v_rows``: existing uint8 storage [pages, kv_heads, page_tokens, row bytes]."""

    def __init__(self, n_seq: int, max_seq: int, kv_heads: int, head_dim: int, page_tokens: int = 0, n_pages: int = 0,
                 page_table=None, k_rows=None, v_rows=None, device=None):
        self.row_bytes = native.load().bt_kv4_row_bytes(head_dim)
        if not self.row_bytes:
            raise ValueError("KV4Cache: head_dim must be 64, 128 or 256")
        if min(n_seq, max_seq, kv_heads) <= 0:
            raise ValueError("KV4Cache: n_seq, max_seq and kv_heads must be positive")
        self.n_seq, self.max_seq, self.kv_heads, self.head_dim = n_seq, max_seq, kv_heads, head_dim
        self.paged = page_tokens > 0
        if (k_rows is None) != (v_rows is None):
            raise ValueError("KV4Cache: give both k_rows and v_rows, or neither")
        device = k_rows.device if k_rows is not None else torch.device("cuda" if device is None else device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        self.page_tokens = page_tokens if self.paged else (max_seq + 15) // 16 * 16
        if k_rows is not None:
            self.n_pages = k_rows.shape[0]
        else:
            self.n_pages = n_pages if self.paged else n_seq
        shape = (self.n_pages, kv_heads, self.page_tokens, self.row_bytes)
        if k_rows is None:
            k_rows, v_rows = (torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2))
        for name, t in (("k_rows", k_rows), ("v_rows", v_rows)):
            if t.dtype != torch.uint8 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != device:
                raise ValueError(f"KV4Cache: {name} must be contiguous uint8 {shape} on {device}")
        self.k_rows, self.v_rows = k_rows, v_rows
        self.max_pages = -(-max_seq // self.page_tokens)
        self._free = self._held = None
        if self.paged:
            if page_table is None:
                page_table = torch.full((n_seq, self.max_pages), -1, dtype=torch.int32, device=device)
                self._free = list(range(self.n_pages - 1, -1, -1))
                self._held = [[] for _ in range(n_seq)]
            if (page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != n_seq
                    or page_table.shape[1] < self.max_pages or not page_table.is_contiguous() or page_table.device != device):
                raise ValueError(f"KV4Cache: page_table must be contiguous int32 [{n_seq}, >= {self.max_pages}] on {device}")
            self.max_pages = page_table.shape[1]
        elif page_table is not None:
            raise ValueError("KV4Cache: a page_table needs page_tokens")
        self.page_table = page_table
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self._c = KV4(k_rows.data_ptr(), v_rows.data_ptr(), page_table.data_ptr() if self.paged else None,
                      self.status.data_ptr(), n_seq, max_seq, kv_heads, head_dim, self.page_tokens, self.n_pages,
                      self.max_pages, 0)
        self._ref = C.addressof(self._c)
        self._index = device.index

    # ------------------------------------------------------------ pages

    def reserve(self, slot: int, positions: int):
        """Pages for positions 0 .. positions - 1 of a slot; MemoryError (and none taken) when too few are free."""
        if self._free is None:
            raise ValueError("reserve: this cache does not hand out its pages")
        if not 0 <= slot < self.n_seq or not 0 <= positions <= self.max_seq:
            raise IndexError("reserve: slot or positions out of range")
        held = self._held[slot]
        more = -(-positions // self.page_tokens) - len(held)
        if more <= 0:
            return
        if more > len(self._free):
            raise MemoryError(f"reserve: {more} pages needed, {len(self._free)} free")
        new = [self._free.pop() for _ in range(more)]
        self.page_table[slot, len(held):len(held) + more] = torch.tensor(new, dtype=torch.int32, device=self.device)
        held += new

    def release(self, slot: int):
        """A slot's pages back to the pool.  Work that reads them has to be on the same stream, or done."""
        if self._free is None:
            raise ValueError("release: this cache does not hand out its pages")
        if not 0 <= slot < self.n_seq:
            raise IndexError("release: slot out of range")
        self._free += reversed(self._held[slot])
        self._held[slot] = []
        self.page_table[slot] = -1

    def pages(self):
        """(free, total) pages of the pool."""
        return (len(self._free) if self._free is not None else 0), self.n_pages

    def check(self):
        """Waits for the device (all of its streams) and raises IndexError if a call met a slot, position, length
        or page out of range since the last check, CudaBackendError if a device wait gave up."""
        if self.device.type == "cuda":
            torch.cuda.synchronize(self.device)
        status = int(self.status.item())
        self.status.zero_()
        if status & native.BT_KV4_TIMEOUT:
            for key in [k for k in _workspaces if k[0] == self._index]:  # (to be cleared before its next call)
                del _workspaces[key]
            raise native.CudaBackendError(native.BT_ERR_DEVICE_TIMEOUT, "KV4Cache: a device wait gave up")
        if status & native.BT_KV4_RANGE:
            raise IndexError("KV4Cache: a slot, position, length or page was out of range")

    def _tensors(self):
        return (self.k_rows, self.v_rows, self.status) + (() if self.page_table is None else (self.page_table,))

    # ------------------------------------------------------------ rows

    def append(self, k, v, slots, positions, stream=None):
        """Stores k, v [T, KVH, hd] at (slots[t], positions[t]); slots < 0: padding."""
        self._append(None, k, v, None, None, slots, positions, None, 0.0, None, stream)

    def append_normed(self, q, k, v, q_weight, k_weight, slots, positions, table, eps: float = 1e-5, q_out=None, stream=None):
        """qk_norm_rope of q and k with the keys and values stored, one launch (bt_cuda_kv4_append); returns
        the queries."""
        return self._append(q, k, v, q_weight, k_weight, slots, positions, table, eps, q_out, stream)

    def _append(self, q, k, v, q_weight, k_weight, slots, positions, table, eps, q_out, stream):
        if stream is not None and _elsewhere(stream):
            return _on_stream(stream, self._tensors(), self._append, q, k, v, q_weight, k_weight, slots, positions, table, eps,
                              q_out, None)
        if k.dim() != 3:
            raise ValueError("append: expected [tokens, kv_heads, head_dim] tensors")
        dev, hd, tokens, dtype = self._index, self.head_dim, k.shape[0], k.dtype
        shape = (tokens, self.kv_heads, hd)  # of the cache
        kh = _heads(k, "k", shape, dtype, dev)
        qh = qoh = _NO_HEADS
        heads = 0
        if q is not None:
            heads = q.shape[1] if q.dim() == 3 else 0
            q_shape = (tokens, heads, hd)
            qh = _heads(q, "q", q_shape, dtype, dev)
            q_out, qoh = _out(q_out, "q_out", q_shape, q, dev)
        a = _pack_qk.pack(*qh, *kh, *_heads(v, "v", shape, dtype, dev), *qoh, *_NO_HEADS,
                          0 if q_weight is None else _vector(q_weight, "q_weight", hd, torch.float32, dev),
                          0 if k_weight is None else _vector(k_weight, "k_weight", hd, torch.float32, dev),
                          _vector(positions, "positions", tokens, torch.int32, dev), _vector(slots, "slots", tokens, torch.int32, dev),
                          *_rope(table, dev), tokens, heads, self.kv_heads, hd, _dtype(k), eps)
        _launch(native.load().bt_cuda_kv4_append, "bt_cuda_kv4_append", dev, self._ref, a)
        return q_out

    def read(self, slots, positions, dtype=torch.float16, stream=None):
        """The values that the rows at (slots[t], positions[t]) stand for: k, v [T, KVH, hd]."""
        if stream is not None and _elsewhere(stream):
            return _on_stream(stream, self._tensors(), self.read, slots, positions, dtype)
        dev, tokens = self._index, positions.numel()
        if dtype not in _DTYPES:
            raise ValueError("read: dtype must be float32, float16 or bfloat16")
        k = torch.empty((tokens, self.kv_heads, self.head_dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        _launch(native.load().bt_cuda_kv4_read, "bt_cuda_kv4_read", dev, self._ref,
                _vector(slots, "slots", tokens, torch.int32, dev), _vector(positions, "positions", tokens, torch.int32, dev),
                tokens, _DTYPES[dtype], k.data_ptr(), v.data_ptr())
        return k, v

    # ------------------------------------------------------------ attention

    def attention(self, q, kv_len, q_start=None, slots=None, max_q: int = 0, window: int = 0, sinks: int = 0,
                  scale: float | None = None, out=None, stream=None):
        """Causal attention of q [T, H, hd] over the cache (bt_cuda_kv4_attention), with an optional sliding
        window whose first ``sinks`` positions stay visible.

        kv_len [n] int32: cached positions of each sequence; its queries are the last ones.  q_start
        [n + 1] int32: sequence i's queries are rows q_start[i] .. q_start[i + 1] - 1 of q; None: one each.
        slots [n] int32: the sequences' slots; None: sequence i is slot i.  max_q: no sequence has more
        queries (0: not known).  Rows of q that belong to no sequence are not written (in a new output they
        hold anything).  16-bit queries are answered with fp16 operands inside (errors in bt_cuda.h), fp32 ones
        to fp32's precision, at several times the cost where rows are many."""
        if stream is not None and _elsewhere(stream):
            return _on_stream(stream, self._tensors(), self.attention, q, kv_len, q_start, slots, max_q, window, sinks, scale, out)
        qh = _heads(q, "q")
        dev, shape, n = self._index, q.shape, kv_len.numel()
        tokens, heads, hd = shape
        if hd != self.head_dim or q.get_device() != dev:
            raise ValueError("attention: q must have the cache's head_dim and device")
        if min(window, sinks, max_q) < 0 or max(window, sinks, max_q) > 0xffffffff:
            raise ValueError("attention: window, sinks and max_q must be in 0 .. 2^32 - 1")
        if scale is None:
            scale = hd ** -0.5
        elif not abs(scale) < 2e38:
            raise ValueError("attention: scale is not finite")
        out, oh = _out(out, "out", shape, q, dev)
        a = _pack_attn.pack(*qh, *oh, _vector(kv_len, "kv_len", n, torch.int32, dev),
                            0 if q_start is None else _vector(q_start, "q_start", n + 1, torch.int32, dev),
                            0 if slots is None else _vector(slots, "slots", n, torch.int32, dev),
                            n, tokens, heads, max_q, window, sinks, _dtype(q), scale)
        lib, s, here = native.load(), _raw_stream(dev), dev == _current_device()
        capture, cache = 0, _workspaces
        if not here or _is_capturing():
            capture = lib.bt_cuda_capture_id(s)
            cache = _captured if capture else _workspaces
        ws = cache.get((dev, s))
        if ws is None or ws[3] != capture:
            ws = _new_workspace(cache, dev, s, capture)
        if here:
            rc = lib.bt_cuda_kv4_attention(self._ref, a, ws[0], ws[1], s)
        else:
            with torch.cuda.device(dev):
                rc = lib.bt_cuda_kv4_attention(self._ref, a, ws[0], ws[1], s)
        if rc:
            native.check(rc, "bt_cuda_kv4_attention")
        return out


def sample_batch(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, token=None, logprob=None, stream=None):
    """A token for every row of logits [B, V] from the given random numbers u [B] in [0, 1)
    (bt_cuda_sample_batch).  temperature, top_p, min_p [B] float32 and top_k [B] int32 on the device, or
    None for none of that.  Returns (token [B] int32, logprob [B] float32)."""
    if stream is not None and _elsewhere(stream):
        return _on_stream(stream, (), sample_batch, logits, u, temperature, top_k, top_p, min_p, token, logprob)
    if logits.dim() != 2 or not logits.is_cuda or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("sample_batch: expected a [rows, vocab] CUDA tensor with contiguous rows")
    dev, (rows, vocab) = logits.get_device(), logits.shape
    f32, i32 = torch.float32, torch.int32
    token = torch.empty(rows, dtype=i32, device=logits.device) if token is None else token
    logprob = torch.empty(rows, dtype=f32, device=logits.device) if logprob is None else logprob
    a = _pack_sample.pack(logits.data_ptr(), logits.stride(0), _vector(u, "u", rows, f32, dev),
                          0 if temperature is None else _vector(temperature, "temperature", rows, f32, dev),
                          0 if top_k is None else _vector(top_k, "top_k", rows, i32, dev),
                          0 if top_p is None else _vector(top_p, "top_p", rows, f32, dev),
                          0 if min_p is None else _vector(min_p, "min_p", rows, f32, dev),
                          _vector(token, "token", rows, i32, dev), _vector(logprob, "logprob", rows, f32, dev),
                          rows, vocab, _dtype(logits), 0)
    _launch(native.load().bt_cuda_sample_batch, "bt_cuda_sample_batch", dev, a)
    return token, logprob
