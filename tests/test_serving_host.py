"""CPU: the serving operators' refusals, struct layouts and the page bookkeeping of KV4Cache's C side
(argument checks return before anything reaches a device)."""
import ctypes as C
import re

import pytest

from conftest import ROOT


@pytest.fixture(scope="module")
def nat():
    from blocktensor_b200 import native
    native.load()
    return native


def kv4(nat, **kw):
    """A well-formed contiguous cache descriptor (addresses that are never read)."""
    f = dict(k_rows=4096, v_rows=8192, page_table=None, status=None, n_seq=2, max_seq=100, kv_heads=2, head_dim=128,
             page_tokens=112, n_pages=2, max_pages=1, reserved=0)
    f.update(kw)
    return nat.KV4(**f)


def qk(nat, **kw):
    f = dict(q=4096, q_token_stride=512, q_head_stride=128, k=4096, k_token_stride=256, k_head_stride=128, v=4096,
             v_token_stride=256, v_head_stride=128, q_out=4096, q_out_token_stride=512, q_out_head_stride=128, k_out=4096,
             k_out_token_stride=256, k_out_head_stride=128, positions=4096, slots=4096, rope=4096, rope_positions=100,
             rot_dim=128, tokens=3, heads=4, kv_heads=2, head_dim=128, dtype=0, eps=1e-5)
    f.update(kw)
    return nat.QkArgs(**f)


def refused(nat, name, *args, match):
    with pytest.raises(ValueError, match=match):
        nat.call(name, *args)


def test_row_bytes(nat):
    lib = nat.load()
    assert [lib.bt_kv4_row_bytes(h) for h in (64, 128, 256)] == [36, 72, 144]
    assert [lib.bt_kv4_row_bytes(h) for h in (0, 32, 96, 512)] == [0, 0, 0, 0]


def test_struct_sizes(nat):
    """The ctypes structs are as wide as the header's members say (8-byte pointers and strides, 4-byte rest)."""
    src = open(f"{ROOT}/include/bt_cuda.h").read()
    wide = {"bt_heads": 24}
    for name, cls in (("bt_kv4", nat.KV4), ("bt_qk_args", nat.QkArgs), ("bt_kv4_attn_args", nat.KV4AttnArgs),
                      ("bt_sample_args", nat.SampleArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), src, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        total = 0
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            n = decl.count(",") + 1
            size = wide["bt_heads"] if decl.startswith("bt_heads") else 8 if "*" in decl or "int64" in decl else 4
            total += n * size
        assert (total + 7) // 8 * 8 == C.sizeof(cls), name


@pytest.mark.parametrize("kw,match", [
    (dict(k_rows=None), "null cache rows"), (dict(v_rows=8193), "16-byte aligned"), (dict(head_dim=96), "head_dim"),
    (dict(kv_heads=0), "kv_heads"), (dict(n_seq=0), "n_seq"), (dict(max_seq=0), "max_seq"),
    (dict(page_tokens=100), "page_tokens"), (dict(page_tokens=96), "page_tokens"), (dict(n_pages=3), "n_pages"),
    (dict(page_table=4096, page_tokens=48), "power of two"), (dict(page_table=4096, page_tokens=8), "power of two"),
    (dict(page_table=4096, page_tokens=64, max_pages=1), "less than max_seq"),
    (dict(page_table=4096, page_tokens=64, max_pages=2, n_pages=0), "pages"),
])
def test_cache_refusals(nat, kw, match):
    c = kv4(nat, **kw)
    refused(nat, "bt_cuda_kv4_read", C.byref(c), 4096, 4096, 1, 0, 4096, 4096, None, match=match)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "dtype"), (dict(head_dim=80), "head_dim"), (dict(rot_dim=24), "rot_dim"), (dict(rot_dim=144), "rot_dim"),
    (dict(rot_dim=0), "rot_dim"), (dict(positions=None), "positions"), (dict(q_out=None), "q_out"), (dict(k_out=None), "k_out"),
    (dict(q=None, k=None), "nothing"), (dict(q_weight=4098), "aligned"), (dict(rope=4100), "aligned"), (dict(q=4097), "aligned"),
    (dict(heads=0), "heads"),
])
def test_norm_refusals(nat, kw, match):
    refused(nat, "bt_cuda_qk_norm_rope", C.byref(qk(nat, **kw)), None, match=match)


@pytest.mark.parametrize("kw,match", [
    (dict(kv_heads=4), "cache's"), (dict(head_dim=64), "cache's"), (dict(slots=None), "slots"), (dict(v=None), "values"),
])
def test_append_refusals(nat, kw, match):
    refused(nat, "bt_cuda_kv4_append", C.byref(kv4(nat)), C.byref(qk(nat, **kw)), None, match=match)
    refused(nat, "bt_cuda_kv4_append", None, C.byref(qk(nat)), None, match="null cache")


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=-1), "dtype"), (dict(heads=3), "multiple"), (dict(heads=0), "multiple"), (dict(tokens=3), "one query"),
    (dict(n=5, tokens=5), "more sequences"), (dict(kv_len=None), "null"), (dict(out=None), "null"), (dict(q=4097), "aligned"),
])
def test_attention_refusals(nat, kw, match):
    f = dict(q=4096, q_token_stride=512, q_head_stride=128, out=4096, out_token_stride=512, out_head_stride=128, kv_len=4096,
             q_start=None, slots=None, n=2, tokens=2, heads=4, max_q=0, window=0, sinks=0, dtype=0, scale=0.1)
    f.update(kw)
    refused(nat, "bt_cuda_kv4_attention", C.byref(kv4(nat)), C.byref(nat.KV4AttnArgs(**f)), 4096, 1 << 40, None, match=match)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=7), "dtype"), (dict(logits=None), "null"), (dict(u=None), "null"), (dict(token=None), "null"),
    (dict(vocab=0), "vocab"), (dict(vocab=1 << 23), "vocab"), (dict(logits=4098), "aligned"),
])
def test_sample_refusals(nat, kw, match):
    f = dict(logits=4096, row_stride=100, u=4096, temperature=None, top_k=None, top_p=None, min_p=None, token=4096, logprob=None,
             rows=1, vocab=100, dtype=0, reserved=0)
    f.update(kw)
    refused(nat, "bt_cuda_sample_batch", C.byref(nat.SampleArgs(**f)), None, match=match)


def test_nothing_to_do(nat):
    """No tokens, no rows: success without a launch."""
    before = nat.load().bt_cuda_launch_count()
    nat.call("bt_cuda_qk_norm_rope", C.byref(qk(nat, tokens=0)), None)
    nat.call("bt_cuda_kv4_append", C.byref(kv4(nat)), C.byref(qk(nat, tokens=0)), None)
    nat.call("bt_cuda_kv4_read", C.byref(kv4(nat)), None, None, 0, 0, None, None, None)
    nat.call("bt_cuda_sample_batch", C.byref(nat.SampleArgs(rows=0)), None)
    assert nat.load().bt_cuda_launch_count() == before


def test_page_bookkeeping():
    """reserve / release on host tensors: pages taken in order, returned, and none taken when too few are free."""
    import blocktensor_b200 as bt
    c = bt.KV4Cache(3, 100, 2, 64, page_tokens=16, n_pages=8, device="cpu")
    assert c.pages() == (8, 8) and c.max_pages == 7
    c.reserve(0, 33)
    c.reserve(1, 16)
    assert c.pages() == (4, 8)
    taken = c.page_table[0, :3].tolist() + c.page_table[1, :1].tolist()
    assert len(set(taken)) == 4 and min(taken) >= 0 and c.page_table[0, 3] == -1
    c.reserve(0, 40)  # still three pages
    assert c.pages() == (4, 8)
    with pytest.raises(MemoryError):
        c.reserve(2, 65)
    assert c.pages() == (4, 8)
    with pytest.raises(IndexError):
        c.reserve(3, 1)
    c.release(0)
    assert c.pages() == (7, 8) and c.page_table[0].eq(-1).all()
    with pytest.raises(ValueError):
        bt.KV4Cache(3, 100, 2, 64, device="cpu").reserve(0, 1)


@pytest.mark.parametrize("kw", [
    dict(head_dim=48), dict(n_seq=0), dict(page_table="x"), dict(k_rows="x"), dict(page_tokens=16, n_pages=4, page_table="y"),
])
def test_cache_object_refusals(kw):
    import torch
    import blocktensor_b200 as bt
    if kw.get("page_table") == "x":
        kw["page_table"] = torch.zeros(3, 7, dtype=torch.int32)
    if kw.get("page_table") == "y":
        kw["page_table"] = torch.zeros(3, 6, dtype=torch.int32)  # too narrow for 100 positions
    if kw.get("k_rows") == "x":
        kw["k_rows"] = torch.zeros(3, 2, 112, 36, dtype=torch.uint8)  # without v_rows
    args = dict(n_seq=3, max_seq=100, kv_heads=2, head_dim=64, device="cpu")
    args.update(kw)
    with pytest.raises(ValueError):
        bt.KV4Cache(**args)


def test_workspace_constants(nat):
    """The bindings' constants are the header's; a library without a device reports no workspace and no capture."""
    src = open(f"{ROOT}/include/bt_cuda.h").read()
    assert int(re.search(r"#define BT_KV4_WORKSPACE_ZERO (\d+)u", src).group(1)) == nat.BT_KV4_WORKSPACE_ZERO
    assert nat.load().bt_cuda_capture_id(None) == 0
    refused(nat, "bt_cuda_kv4_inject_stall", 256, match="255")
    nat.call("bt_cuda_kv4_inject_stall", 0)


def test_timeout_drops_the_scratch():
    """What a call whose wait gave up leaves in the attention's scratch serves no later call of that device."""
    import blocktensor_b200 as bt
    from blocktensor_b200 import native, serving
    c = bt.KV4Cache(1, 16, 1, 64, device="cpu")
    keys = [(c._index, 7), (c._index, 9), ("another device", 7)]
    for k in keys:
        serving._workspaces[k] = (0, 0, None, 0)
    try:
        c.status.fill_(native.BT_KV4_RANGE)
        with pytest.raises(IndexError):
            c.check()
        assert all(k in serving._workspaces for k in keys)
        c.status.fill_(native.BT_KV4_TIMEOUT)
        with pytest.raises(native.CudaBackendError) as e:
            c.check()
        assert e.value.code == native.BT_ERR_DEVICE_TIMEOUT
        assert [k in serving._workspaces for k in keys] == [False, False, True]
        c.check()
    finally:
        for k in keys:
            serving._workspaces.pop(k, None)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_attention_scale_refusals(nat, scale):
    """(3e38 passes fp32's range on its way to powers of two)"""
    a = nat.KV4AttnArgs(q=4096, q_token_stride=512, q_head_stride=128, out=4096, out_token_stride=512, out_head_stride=128,
                        kv_len=4096, n=2, tokens=2, heads=4, scale=scale)
    refused(nat, "bt_cuda_kv4_attention", C.byref(kv4(nat)), C.byref(a), 4096, 1 << 40, None, match="finite")


def test_page_slots_out_of_range():
    """A slot that is not the cache's is refused, a negative one too (it names none, not the last)."""
    import blocktensor_b200 as bt
    c = bt.KV4Cache(3, 100, 2, 64, page_tokens=16, n_pages=8, device="cpu")
    c.reserve(2, 33)
    for slot in (-1, 3):
        with pytest.raises(IndexError):
            c.release(slot)
        with pytest.raises(IndexError):
            c.reserve(slot, 1)
    with pytest.raises(IndexError):
        c.reserve(1, -1)
    assert c.pages() == (5, 8) and int((c.page_table[2] >= 0).sum()) == 3
