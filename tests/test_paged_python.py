"""Checks of the paged cache's Python side that need no GPU: stand-ins for device
tensors, which are refused before anything is launched."""
import pytest


class Dev:
    """What m27b looks at of a device tensor."""

    def __init__(self, torch, shape, dtype, dev=0, contiguous=True, grad=False):
        self.t = torch.empty(shape, dtype=dtype, device="meta")
        self.shape, self.dtype, self.is_cuda, self.dev, self.c, self.requires_grad = self.t.shape, dtype, True, dev, contiguous, grad

    def get_device(self):
        return self.dev

    def is_contiguous(self):
        return self.c

    def data_ptr(self):
        return 0x10000

    def __getitem__(self, i):
        return self.t[i]

    def __getattr__(self, name):
        return getattr(self.t, name)


def _attn(torch, m27b, **kw):
    bf, i32 = torch.bfloat16, torch.int32
    dev = lambda *a, **k: Dev(torch, *a, **k)  # noqa: E731
    a = dict(k=dev((4, 16, 2, 64), bf), v=dev((4, 16, 2, 64), bf), table=dev((1, 4), i32), q=dev((3, 4, 64), bf),
             cu_q=dev((2,), i32), lens=dev((1,), i32), out=dev((3, 4, 64), bf),
             scratch=dev((m27b._paged_lib().m27b_paged_attn_scratch_bytes(4, 2, 64),), torch.uint8))
    a.update(kw)
    kv = m27b.PagedKV(a.pop("k"), a.pop("v"), a.pop("table"))
    m27b.paged_attn(kv, **a)


def _torch():
    import torch
    return torch


@pytest.mark.parametrize("shape,contiguous", [((10,), True), ((1 << 26,), False), ((0,), True)])
def test_scratch_that_is_no_memory(m27b, shape, contiguous):
    torch = _torch()
    with pytest.raises(m27b.M27BError, match="scratch"):
        _attn(torch, m27b, scratch=Dev(torch, shape, torch.uint8, contiguous=contiguous))


def _rope(torch, m27b, **kw):
    bf, i32, f32 = torch.bfloat16, torch.int32, torch.float32
    dev = lambda *a, **k: Dev(torch, *a, **k)  # noqa: E731
    a = dict(q=dev((3, 4, 64), f32), k=dev((3, 2, 64), f32), v=dev((3, 2, 64), f32), cu_q=dev((2,), i32), lens=dev((1,), i32),
             rope=dev((10, 32, 2), f32), q_out=dev((3, 4, 64), bf), q_norm=dev((64,), f32), k_norm=dev((64,), f32),
             rows=dev((1,), i32), positions=dev((3,), i32))
    a.update(kw)
    m27b.rope_append(m27b.PagedKV(dev((4, 16, 2, 64), bf), dev((4, 16, 2, 64), bf), dev((1, 4), i32)), **a)


def _pages(torch, m27b, pool=0, ref=0, table=0, lens=0):
    i32 = torch.int32
    return m27b.PageSet(Dev(torch, (3, 4), i32, table), Dev(torch, (8,), i32, ref), Dev(torch, (3,), i32, lens), 16,
                        Dev(torch, (2, 8, 64), torch.bfloat16, pool))


def test_tensors_of_another_device(m27b):
    # the kernels would read or write another GPU's memory through this one's context
    torch = _torch()
    bf, i32, f32 = torch.bfloat16, torch.int32, torch.float32
    one = lambda shape, dt: Dev(torch, shape, dt, dev=1)  # noqa: E731
    size = m27b._paged_lib().m27b_paged_attn_scratch_bytes(4, 2, 64)
    for kw in (dict(k=one((4, 16, 2, 64), bf)), dict(v=one((4, 16, 2, 64), bf)), dict(table=one((1, 4), i32)), dict(q=one((3, 4, 64), bf)),
               dict(cu_q=one((2,), i32)), dict(lens=one((1,), i32)), dict(out=one((3, 4, 64), bf)), dict(rows=one((1,), i32)),
               dict(lse=one((3, 4), f32)), dict(scratch=one((size,), torch.uint8))):
        with pytest.raises(m27b.M27BError, match="on device"):
            _attn(torch, m27b, **kw)
    for kw in (dict(q=one((3, 4, 64), f32)), dict(k=one((3, 2, 64), f32)), dict(v=one((3, 2, 64), f32)), dict(rope=one((10, 32, 2), f32)),
               dict(q_out=one((3, 4, 64), bf)), dict(q_norm=one((64,), f32)), dict(k_norm=one((64,), f32)), dict(cu_q=one((2,), i32)),
               dict(lens=one((1,), i32)), dict(rows=one((1,), i32)), dict(positions=one((3,), i32))):
        with pytest.raises(m27b.M27BError, match="on device"):
            _rope(torch, m27b, **kw)
    for kw in (dict(pool=1), dict(table=1), dict(lens=1)):
        with pytest.raises(m27b.M27BError, match="device"):
            _pages(torch, m27b, **kw)
    ps = _pages(torch, m27b)
    for call in (ps.resize, ps.fork, ps.copy):
        with pytest.raises(m27b.M27BError, match="on device"):
            call(one((1,), i32), Dev(torch, (1,), i32))
        with pytest.raises(m27b.M27BError, match="on device"):
            call(Dev(torch, (1,), i32), one((1,), i32))
    with pytest.raises(m27b.M27BError, match="on device"):
        ps.free(one((1,), i32))
    with pytest.raises(m27b.M27BError, match="on device"):
        ps.compact(n_live=one((1,), i32))


def test_another_current_device_or_stream(m27b, monkeypatch):
    torch = _torch()

    class Stream:
        device_index, cuda_stream = 1, 0

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    for call in (lambda: _attn(torch, m27b), lambda: _rope(torch, m27b), lambda: _pages(torch, m27b).compact()):
        with pytest.raises(m27b.M27BError, match="current device is 1"):
            call()
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    for call in (lambda: _attn(torch, m27b, stream=Stream), lambda: _rope(torch, m27b, stream=Stream)):
        with pytest.raises(m27b.M27BError, match="the stream's 1"):
            call()


def test_tensors_that_require_grad(m27b, monkeypatch):
    # the results would carry no gradient without a word
    torch = _torch()
    bf, f32 = torch.bfloat16, torch.float32
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)  # what no_grad lets through ends at the device
    want = lambda shape, dt: Dev(torch, shape, dt, grad=True)  # noqa: E731
    for call, kw in ((_attn, dict(q=want((3, 4, 64), bf))), (_attn, dict(k=want((4, 16, 2, 64), bf))),
                     (_attn, dict(v=want((4, 16, 2, 64), bf))), (_rope, dict(q=want((3, 4, 64), f32))),
                     (_rope, dict(k=want((3, 2, 64), f32))), (_rope, dict(v=want((3, 2, 64), f32))),
                     (_rope, dict(q_norm=want((64,), f32))), (_rope, dict(k_norm=want((64,), f32)))):
        with pytest.raises(m27b.M27BError, match="no backward pass"):
            call(torch, m27b, **kw)
        with torch.no_grad(), pytest.raises(m27b.M27BError, match="current device"):
            call(torch, m27b, **kw)
