"""Refusals of the paged cache's entries (include/m27b_paged.h): every check is
made on the host before any CUDA call, so no GPU is needed."""
import ctypes

import pytest


def _kv(m, **kw):
    d = dict(k=0x10000, v=0x20000, table=0x30000, type=m.BF16, n_pages=4, page_size=16, n_kv=2, head_dim=128, n_rows=3,
             n_cols=2, page_stride=16 * 2 * 128)
    d.update(kw)
    return m._PagedKV(**d)


def _batch(m, **kw):
    d = dict(cu_q=0x40000, lens=0x50000, rows=None, n_seq=2, n_tok=2)
    d.update(kw)
    return m._PagedBatch.pack(*(v or 0 for v in d.values()))


BAD_KV = [(dict(k=None), "null pool"), (dict(table=None), "null pool"), (dict(v=0x20008), "16-byte"), (dict(type=0), "f16 or bf16"),
          (dict(page_size=24), "page_size"), (dict(page_size=8), "page_size"), (dict(page_size=512), "page_size"),
          (dict(head_dim=96), "head_dim"), (dict(n_kv=0), "n_kv"), (dict(n_pages=0), "empty"), (dict(n_cols=0), "empty"),
          (dict(page_stride=4095), "page_stride"), (dict(page_stride=4100), "page_stride"),
          (dict(n_cols=1 << 30), "31 bits"), (dict(page_stride=1 << 61), "too large")]
BAD_BATCH = [(dict(cu_q=None), "null batch"), (dict(lens=None), "null batch"), (dict(n_seq=-1), "n_seq"),
             (dict(n_tok=-1), "n_tok"), (dict(n_seq=4), "table rows")]


def _attn(m, kv=None, bt=None, q=0x60000, qs=512, n_q=4, scale=1.0, window=0, out=0x70000, os=512, scr=0x80000):
    m._paged_lib()
    return m.call_raw("m27b_paged_attn", ctypes.byref(kv or _kv(m)), bt or _batch(m), q, qs, n_q, scale,
                      window, out, os, None, scr, None)


@pytest.mark.parametrize("kw,needle", BAD_KV)
def test_bad_cache(m27b, kw, needle):
    ok, msg = _attn(m27b, kv=_kv(m27b, **kw))
    assert not ok and needle in msg, msg


@pytest.mark.parametrize("kw,needle", BAD_BATCH)
def test_bad_batch(m27b, kw, needle):
    ok, msg = _attn(m27b, bt=_batch(m27b, **kw))
    assert not ok and needle in msg, msg


@pytest.mark.parametrize("kw,needle", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(scr=None), "null"), (dict(q=0x60008), "16-byte"),
    (dict(n_q=3), "multiple of n_kv"), (dict(n_q=258), "at most 128"), (dict(qs=256), "strides"), (dict(qs=516), "strides"),
    (dict(os=504), "strides"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale")])
def test_bad_attention(m27b, kw, needle):
    ok, msg = _attn(m27b, **kw)
    assert not ok and needle in msg, msg


def test_nothing_to_attend_is_no_error(m27b):
    assert _attn(m27b, bt=_batch(m27b, n_seq=0)) == (True, "")
    assert _attn(m27b, bt=_batch(m27b, n_tok=0)) == (True, "")


def test_scratch_sizes(m27b):
    L = m27b._paged_lib()
    assert L.m27b_paged_attn_scratch_bytes(24, 4, 256) > 0
    for bad in ((0, 1, 128), (3, 2, 128), (129, 1, 128), (4, 2, 96), (4, 0, 128)):
        assert L.m27b_paged_attn_scratch_bytes(*bad) == 0
    assert L.m27b_pages_scratch_bytes(100, 5, 7) >= 4 * (3 * 100 + 5)
    assert L.m27b_pages_scratch_bytes(0, 5, 7) == L.m27b_pages_scratch_bytes(4, 0, 7) == L.m27b_pages_scratch_bytes(4, 4, -1) == 0


def _rope(m, kv=None, rope=None, heads=None, out=0x90000, os=512):
    m._paged_lib()
    r = dict(table=0xa0000, n_pos=10, n_rot=64, interleaved=0, positions=None)
    r.update(rope or {})
    h = dict(q=0x60000, k=0x61000, v=0x62000, q_stride=1024, k_stride=1024, v_stride=1024, src_type=m.F32, n_q=4,
             q_norm=None, k_norm=None, eps=1e-6)
    h.update(heads or {})
    return m.call_raw("m27b_rope_append", ctypes.byref(kv or _kv(m)), _batch(m), m._Rope.pack(*(v or 0 for v in r.values())),
                      m._Heads.pack(*(v or 0 for v in h.values())), out, os, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(rope=dict(table=None)), "rope table"), (dict(rope=dict(table=0xa0008)), "rope table"), (dict(rope=dict(n_rot=8)), "n_rot"),
    (dict(rope=dict(n_rot=144)), "n_rot"), (dict(rope=dict(n_rot=40)), "n_rot"), (dict(rope=dict(n_pos=0)), "n_rot"),
    (dict(heads=dict(k=None)), "null k"), (dict(heads=dict(q=None)), "null q"), (dict(out=None), "null q"),
    (dict(heads=dict(n_q=-1)), "n_q"), (dict(heads=dict(src_type=1)), "cache's type"), (dict(heads=dict(k=0x61004)), "16-byte"),
    (dict(heads=dict(q_norm=0x100004)), "16-byte"), (dict(heads=dict(q_stride=1022)), "16 bytes"),
    (dict(heads=dict(v_stride=128)), "shorter"), (dict(os=256), "shorter"), (dict(out=0x60000), "may be q"),
    (dict(kv=dict(page_size=5)), "page_size")])
def test_bad_rope(m27b, kw, needle):
    kw = dict(kw)
    if "kv" in kw:
        kw["kv"] = _kv(m27b, **kw["kv"])
    ok, msg = _rope(m27b, **kw)
    assert not ok and needle in msg, msg


@pytest.mark.parametrize("args,needle", [
    ((None, 4, 64, 1e4, None), "aligned"), ((0x1004, 4, 64, 1e4, None), "aligned"), ((0x1000, 0, 64, 1e4, None), "n_pos"),
    ((0x1000, 4, 63, 1e4, None), "even"), ((0x1000, 4, 64, 0.0, None), "theta"), ((0x1000, 4, 64, 1e4, dict(kind=3)), "unknown"),
    ((0x1000, 4, 64, 1e4, dict(kind=1, factor=0.5)), "factor"), ((0x1000, 4, 64, 1e4, dict(kind=2, factor=2.0)), "yarn")])
def test_bad_rope_table(m27b, args, needle):
    m27b._paged_lib()
    s = ctypes.byref(m27b._RopeScaling(**args[4])) if args[4] else None
    ok, msg = m27b.call_raw("m27b_rope_table", *args[:4], s, None)
    assert not ok and needle in msg, msg


def _pages(m, **kw):
    d = dict(ref=0x1000, table=0x2000, lens=0x3000, n_pages=8, page_size=16, n_rows=4, n_cols=4)
    d.update(kw)
    return m._Pages(**d)


def _pool(m, **kw):
    d = dict(base=0x10000, n_planes=2, plane_stride=1024, page_stride=64, page_bytes=64)
    d.update(kw)
    return (m._PagePool * 1)(m._PagePool(**d))


@pytest.mark.parametrize("pages,pool,n_pools,n,scr,needle", [
    (dict(ref=None), {}, 1, 1, 0x5000, "null"), (dict(n_rows=0), {}, 1, 1, 0x5000, "empty"), (dict(page_size=0), {}, 1, 1, 0x5000, "page_size"),
    (dict(n_pages=1 << 27), {}, 1, 1, 0x5000, "2^26"), ({}, dict(base=None), 1, 1, 0x5000, "empty"), ({}, dict(page_bytes=60), 1, 1, 0x5000, "16"),
    ({}, dict(page_stride=48), 1, 1, 0x5000, "shorter"), ({}, {}, 0, 1, 0x5000, "pools"), ({}, {}, 3, 1, 0x5000, "pools"),
    ({}, {}, 1, -1, 0x5000, "bad n"), ({}, {}, 1, 1, None, "scratch"), ({}, {}, 1, 1, 0x5008, "scratch")])
def test_bad_pages(m27b, pages, pool, n_pools, n, scr, needle):
    m27b._paged_lib()
    for name in ("m27b_pages_fork", "m27b_pages_resize"):
        ok, msg = m27b.call_raw(name, ctypes.byref(_pages(m27b, **pages)), _pool(m27b, **pool), n_pools, 0x6000, 0x7000, n, scr,
                                0x8000, None)
        assert not ok and needle in msg, msg
    if n >= 0:
        ok, msg = m27b.call_raw("m27b_pages_compact", ctypes.byref(_pages(m27b, **pages)), _pool(m27b, **pool), n_pools, None, scr, None)
        assert not ok and needle in msg, msg


def test_bad_page_requests(m27b):
    m27b._paged_lib()
    pg, pool = _pages(m27b), _pool(m27b)
    ok, msg = m27b.call_raw("m27b_pages_fork", ctypes.byref(pg), pool, 1, None, 0x7000, 1, 0x5000, 0x8000, None)
    assert not ok and "null requests" in msg
    ok, msg = m27b.call_raw("m27b_pages_free", ctypes.byref(pg), None, 1, None)
    assert not ok and "null rows" in msg
    ok, msg = m27b.call_raw("m27b_pages_copy", pool, 1, 0, 0x1000, 0x2000, 1, None)
    assert not ok and "bad n" in msg
    assert m27b.call_raw("m27b_pages_free", ctypes.byref(pg), None, 0, None) == (True, "")
    assert m27b.call_raw("m27b_pages_fork", ctypes.byref(pg), pool, 1, None, None, 0, 0x5000, None, None) == (True, "")


def test_python_checks_tensors(m27b):
    import torch
    cpu = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(m27b.M27BError, match="on the device"):
        m27b.PagedKV(cpu, cpu, torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(m27b.M27BError, match="one type and layout"):
        m27b.PagedKV(cpu, cpu[:1], torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(m27b.M27BError, match="unsupported heads"):
        m27b.paged_attn_scratch(3, 2, 64, device="cpu")
    with pytest.raises(m27b.M27BError, match="int32 device"):
        m27b._int32(torch.zeros(1, dtype=torch.int64), "rows")
