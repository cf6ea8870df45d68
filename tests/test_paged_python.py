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
