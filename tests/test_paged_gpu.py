"""The paged cache's operators on the GPU (include/m27b_paged.h) against plain
64-bit restatements (tests/_paged_ref.py).

Tolerances.  u is the relative size of half a unit in the last place of the
cache's type: 2^-8 for bf16's 8 significant bits, 2^-11 for f16's 11.
  * rope_append: one rounding of the result, u |x|, and fp32 arithmetic, a few
    2^-24 of the head's largest value: 2e-6 of it.
  * attention: the result's rounding, u |o|; the weights' rounding before the
    product with V, at most u sum p |v|; the scores' fp32 sums, at most ds =
    2^-19 of the largest scale * sum |q||k| of the row, plus 1e-6 for the
    exponential, which change each weight by a relative 2 ds: 2 ds sum p |v|.
    lse: ds + 1e-6 (1 + |lse|).
  * pages: integers and copies, equal."""
import random

import numpy as np
import pytest

import _paged_ref as P

pytestmark = pytest.mark.gpu


def _dt(torch, name):
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def _np(t):
    return t.detach().double().cpu().numpy()


class Cache:
    """Pools filled with noise (NaN and inf past each sequence's end), each sequence's pages anywhere."""

    def __init__(self, torch, m27b, lens, ps, n_kv, hd, dtype, seed, spare=3, pad=0, rows=None, poison=True):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rng = random.Random(seed)
        dt = _dt(torch, dtype)
        held = [P.cdiv(n, ps) for n in lens]
        n_pages = sum(held) + spare
        self.buf = [torch.randn(n_pages, ps * n_kv * hd + pad, generator=g, device="cuda").to(dt) for _ in range(2)]
        self.k, self.v = (b[:, :ps * n_kv * hd].view(n_pages, ps, n_kv, hd) if not pad else
                          b.as_strided((n_pages, ps, n_kv, hd), (b.stride(0), n_kv * hd, hd, 1)) for b in self.buf)
        order = list(range(n_pages))
        rng.shuffle(order)
        self.rows = list(range(len(lens))) if rows is None else rows
        n_rows = max(self.rows, default=0) + 1
        tab = np.full((n_rows, max(held + [1]) + 1), -1, dtype=np.int32)
        ln = np.zeros(n_rows, dtype=np.int32)
        at = 0
        for r, n, h in zip(self.rows, lens, held):
            tab[r, :h] = order[at:at + h]
            ln[r] = n
            at += h
            if n % ps and poison:
                self.k[tab[r, h - 1], n % ps:] = float("nan")
                self.v[tab[r, h - 1], n % ps:] = float("inf")
        for p in order[at:]:
            self.k[p], self.v[p] = float("inf"), float("nan")
        self.tab, self.ln, self.ps, self.lens_list = tab, ln, ps, lens
        self.table = torch.from_numpy(tab).cuda()
        self.lens = torch.from_numpy(ln).cuda()
        self.rows_t = None if rows is None else torch.tensor(rows, dtype=torch.int32, device="cuda")
        self.kv = m27b.PagedKV(self.k, self.v, self.table)

    def seq(self, b):
        """(keys, values) of sequence b, fp64"""
        r, n = self.rows[b], self.lens_list[b]
        ids = self.tab[r, :P.cdiv(n, self.ps)].astype(np.int64)
        import torch
        t = torch.from_numpy(ids).cuda()
        return tuple(_np(x[t]).reshape(-1, *x.shape[2:])[:n] for x in (self.k, self.v))


def _cu(torch, q_lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32, device="cuda")


def _check_attn(torch, m27b, q_lens, kv_lens, n_q, n_kv, hd, dtype, ps, window=0, seed=0, scale=None, lse=True, pad=0,
                rows=None, q_gain=1.0, strided=False):
    c = Cache(torch, m27b, kv_lens, ps, n_kv, hd, dtype, seed, pad=pad, rows=rows)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    total = sum(q_lens)
    wide = torch.randn(total, n_q + 2, hd, generator=g, device="cuda").mul_(q_gain).to(_dt(torch, dtype))
    q = wide[:, 1:1 + n_q] if strided else wide[:, :n_q].contiguous()
    out_w = torch.full((total, n_q + (3 if strided else 0), hd), 7.0, device="cuda").to(q.dtype)
    out = out_w[:, :n_q]
    ls = torch.full((total, n_q), 7.0, device="cuda") if lse else None
    scr = m27b.paged_attn_scratch(n_q, n_kv, hd)
    scr.fill_(255)
    for _ in range(2):  # the scratch may hold anything
        m27b.paged_attn(c.kv, q, _cu(torch, q_lens), c.lens, out, scr, scale=scale, window=window, lse=ls, rows=c.rows_t)
    torch.cuda.synchronize()
    sc, u = hd ** -0.5 if scale is None else scale, P.U[dtype]
    got, got_l, qn, at = _np(out), _np(ls) if lse else None, _np(q), 0
    for b, n in enumerate(q_lens):
        o, l, mag, big = P.attend(qn[at:at + n], *c.seq(b), sc, window)
        ds = 2.0 ** -19 * big + 1e-6
        tol = u * np.abs(o) + (u + 2 * ds[..., None]) * mag * 1.02 + 1e-7
        err = np.abs(got[at:at + n] - o)
        assert np.isfinite(got[at:at + n]).all(), b
        assert (err <= tol).all(), (b, float((err / np.maximum(tol, 1e-30)).max()))
        if lse:
            gl = got_l[at:at + n]
            assert np.array_equal(np.isinf(gl), np.isinf(l)), b
            f = np.isfinite(l)
            assert (np.abs(gl[f] - l[f]) <= (ds + 1e-6 * (1 + np.abs(l)))[f]).all(), b
        at += n
    if strided:
        assert (_np(out_w)[:, n_q:] == 7.0).all()
    assert m27b.device_status() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd,n_q,n_kv", [(256, 24, 4), (128, 16, 8), (64, 8, 1)])
def test_attn_one_token(torch, m27b, dtype, hd, n_q, n_kv):
    _check_attn(torch, m27b, [1] * 9, [1, 2, 15, 16, 17, 63, 64, 65, 1000], n_q, n_kv, hd, dtype, 16, seed=1)


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attn_page_sizes_ragged(torch, m27b, hd, ps):
    _check_attn(torch, m27b, [3, 1, 40, 7, 130], [3, 257, 300, 129, 130], 6, 2, hd, "bf16", ps, seed=2)


@pytest.mark.parametrize("n_q,n_kv", [(1, 1), (5, 1), (7, 7), (64, 1), (128, 1), (12, 4), (33, 3), (256, 2)])
def test_attn_head_groups(torch, m27b, n_q, n_kv):
    _check_attn(torch, m27b, [1, 5, 2], [70, 201, 2], n_q, n_kv, 64, "f16", 16, seed=3)


@pytest.mark.parametrize("window", [1, 2, 16, 64, 65, 100, 127, 129, 1000])
@pytest.mark.parametrize("hd", [128, 256])
def test_attn_window(torch, m27b, window, hd):
    _check_attn(torch, m27b, [1, 70, 33], [500, 400, 33], 6, 2, hd, "bf16", 32, window=window, seed=4)


def test_attn_empty_rows_and_idle_sequences(torch, m27b):
    # no positions at all; fewer positions than tokens; no tokens; one of each
    _check_attn(torch, m27b, [4, 0, 9, 1, 0, 1], [0, 33, 5, 1, 0, 0], 8, 2, 128, "bf16", 16, seed=5)
    _check_attn(torch, m27b, [300, 2], [100, 0], 8, 2, 256, "f16", 16, window=3, seed=6)


def test_attn_no_sequences(torch, m27b):
    c = Cache(torch, m27b, [5], 16, 2, 64, "bf16", 0)
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    m27b.paged_attn(c.kv, q, _cu(torch, []), c.lens, q.clone(), m27b.paged_attn_scratch(4, 2, 64))
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, 5.0)
    m27b.paged_attn(c.kv, q, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), c.lens, out,
                    m27b.paged_attn_scratch(4, 2, 64))
    assert (out[1:] == 5.0).all() and not (out[0] == 5.0).any()  # rows of no sequence are left alone


@pytest.mark.parametrize("dtype,hd,n_q,n_kv", [("bf16", 256, 24, 4), ("f16", 128, 16, 8)])
def test_attn_long_split(torch, m27b, dtype, hd, n_q, n_kv):
    _check_attn(torch, m27b, [1, 2], [9001, 5003], n_q, n_kv, hd, dtype, 64, seed=7)


def test_attn_chunk_on_long_context(torch, m27b):
    _check_attn(torch, m27b, [150], [2001], 6, 1, 256, "bf16", 64, seed=8)
    _check_attn(torch, m27b, [257], [700], 4, 2, 128, "f16", 32, seed=9)


@pytest.mark.parametrize("gain", [0.0, 8.0, 40.0])
def test_attn_flat_and_sharp_softmax(torch, m27b, gain):
    _check_attn(torch, m27b, [1, 33], [777, 333], 6, 2, 128, "bf16", 16, seed=10, q_gain=gain)


def test_attn_rising_scores(torch, m27b):
    # every later position scores higher than all before it: the running maximum moves at every tile
    for hd in (64, 128, 256):
        n, ps = 700, 16
        c = Cache(torch, m27b, [n], ps, 1, hd, "bf16", 11)
        ids = torch.from_numpy(c.tab[0, :P.cdiv(n, ps)].astype(np.int64)).cuda()
        ramp = torch.arange(len(ids) * ps, device="cuda").view(-1, ps, 1).float() / 700
        c.k[ids] = ramp[..., None].expand(-1, -1, 1, hd).to(torch.bfloat16)
        q = torch.ones(5, 2, hd, dtype=torch.bfloat16, device="cuda")
        out, lse = torch.empty_like(q), torch.empty(5, 2, device="cuda")
        m27b.paged_attn(c.kv, q, _cu(torch, [5]), c.lens, out, m27b.paged_attn_scratch(2, 1, hd), scale=1.0, lse=lse)
        o, l, mag, big = P.attend(_np(q), *c.seq(0), 1.0, 0)
        ds = 2.0 ** -19 * big + 1e-6
        u = P.U["bf16"]
        assert (np.abs(_np(out) - o) <= u * np.abs(o) + (u + 2 * ds[..., None]) * mag * 1.02 + 1e-7).all()
        assert (np.abs(_np(lse) - l) <= ds + 1e-6 * (1 + np.abs(l))).all()


def test_attn_strides_rows_and_shared_pages(torch, m27b):
    _check_attn(torch, m27b, [2, 5, 1], [40, 100, 17], 6, 2, 128, "bf16", 16, seed=12, pad=64, rows=[4, 0, 2], strided=True)
    _check_attn(torch, m27b, [1, 66], [40, 100], 6, 2, 256, "f16", 32, seed=13, pad=8, rows=[1, 5], strided=True, scale=0.3)
    # two rows of one cache hold the same pages
    c = Cache(torch, m27b, [90], 16, 2, 64, "bf16", 14)
    tab = c.table.repeat(2, 1).contiguous()
    lens = torch.tensor([90, 64], dtype=torch.int32, device="cuda")
    kv = m27b.PagedKV(c.k, c.v, tab)
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    out = torch.empty_like(q)
    m27b.paged_attn(kv, q, _cu(torch, [1, 1]), lens, out, m27b.paged_attn_scratch(4, 2, 64))
    k, v = c.seq(0)
    for b, n in enumerate((90, 64)):
        o, _, mag, _ = P.attend(_np(q)[b:b + 1], k[:n], v[:n], 0.125, 0)
        assert (np.abs(_np(out)[b] - o[0]) <= 2.0 ** -8 * (np.abs(o[0]) + 1.1 * mag[0]) + 1e-6).all()


def test_attn_many_sequences(torch, m27b):
    rng = random.Random(15)
    n = 700
    q = [rng.choice([0, 1, 1, 1, 2]) for _ in range(n)]
    kv = [x + rng.randrange(0, 90) for x in q]
    _check_attn(torch, m27b, q, kv, 4, 2, 64, "f16", 16, seed=16)


def test_attn_result_does_not_depend_on_the_run(torch, m27b):
    c = Cache(torch, m27b, [5000, 77, 3000], 16, 4, 128, "bf16", 17)
    q = torch.randn(12, 24, 128, device="cuda").bfloat16()
    cu, scr = _cu(torch, [1, 10, 1]), m27b.paged_attn_scratch(24, 4, 128)
    outs = []
    for _ in range(10):
        out = torch.empty_like(q)
        m27b.paged_attn(c.kv, q, cu, c.lens, out, scr)
        outs.append(out)
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_attn_other_stream_and_graph(torch, m27b):
    c = Cache(torch, m27b, [900, 40], 16, 2, 128, "bf16", 18)
    q = torch.randn(2, 8, 128, device="cuda").bfloat16()
    cu, scr = _cu(torch, [1, 1]), m27b.paged_attn_scratch(8, 2, 128)
    want, out = torch.empty_like(q), torch.empty_like(q)
    m27b.paged_attn(c.kv, q, cu, c.lens, want, scr)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    m27b.paged_attn(c.kv, q, cu, c.lens, out, scr, stream=s)
    s.synchronize()
    assert torch.equal(out, want)
    out.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m27b.paged_attn(c.kv, q, cu, c.lens, out, scr)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    # the captured call reads the lengths as they are when it runs
    c.lens.copy_(torch.tensor([333, 40], dtype=torch.int32))
    m27b.paged_attn(c.kv, q, cu, c.lens, want, scr)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# Batches of many rows a sequence run on pairs of CTAs (head_dim 128 and 256).


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("hd,dtype", [(128, "f16"), (256, "bf16")])
def test_attn_many_rows_page_sizes(torch, m27b, hd, dtype, ps):
    _check_attn(torch, m27b, [300, 0, 131, 1], [701, 50, 131, 400], 8, 2, hd, dtype, ps, seed=30)


@pytest.mark.parametrize("window", [1, 63, 100, 128, 129, 500])
@pytest.mark.parametrize("hd", [128, 256])
def test_attn_many_rows_window(torch, m27b, window, hd):
    _check_attn(torch, m27b, [260, 170], [900, 170], 6, 2, hd, "bf16", 32, window=window, seed=31)


@pytest.mark.parametrize("n_q,n_kv", [(1, 1), (128, 1), (7, 1), (10, 5), (64, 1)])
def test_attn_many_rows_head_groups(torch, m27b, n_q, n_kv):
    n = max(3, 600 // (n_q // n_kv))
    _check_attn(torch, m27b, [n, 2 * n], [n + 150, 2 * n], n_q, n_kv, 128, "bf16", 16, seed=32)


def test_attn_many_rows_empty_and_idle(torch, m27b):
    # fewer positions than tokens, none at all, one token, no tokens
    _check_attn(torch, m27b, [400, 90, 0, 300, 1], [150, 0, 77, 300, 513], 8, 2, 128, "f16", 16, seed=33)
    _check_attn(torch, m27b, [257, 3], [100, 0], 12, 2, 256, "bf16", 16, window=40, seed=34)


def test_attn_many_rows_split_runs(torch, m27b):
    # one long item list per kv head: every run begins and ends inside an item
    _check_attn(torch, m27b, [64], [6000], 4, 1, 256, "bf16", 64, seed=35)
    _check_attn(torch, m27b, [700], [1500], 4, 2, 128, "f16", 32, seed=36)


def test_attn_many_rows_strides_and_rows(torch, m27b):
    _check_attn(torch, m27b, [140, 100], [340, 100], 6, 2, 256, "f16", 32, seed=37, pad=8, rows=[3, 1], strided=True, scale=0.2)
    _check_attn(torch, m27b, [200], [333], 8, 2, 128, "bf16", 16, seed=38, pad=64, rows=[2], strided=True)


@pytest.mark.parametrize("gain", [0.0, 8.0, 40.0])
def test_attn_many_rows_flat_and_sharp(torch, m27b, gain):
    _check_attn(torch, m27b, [200], [777], 6, 2, 128, "bf16", 16, seed=39, q_gain=gain)


def test_attn_many_rows_rising_scores(torch, m27b):
    for hd in (128, 256):
        n, ps = 900, 16
        c = Cache(torch, m27b, [n], ps, 1, hd, "bf16", 40)
        ids = torch.from_numpy(c.tab[0, :P.cdiv(n, ps)].astype(np.int64)).cuda()
        ramp = torch.arange(len(ids) * ps, device="cuda").view(-1, ps, 1).float() / 900
        c.k[ids] = ramp[..., None].expand(-1, -1, 1, hd).to(torch.bfloat16)
        q = torch.ones(160, 2, hd, dtype=torch.bfloat16, device="cuda")
        out, lse = torch.empty_like(q), torch.empty(160, 2, device="cuda")
        m27b.paged_attn(c.kv, q, _cu(torch, [160]), c.lens, out, m27b.paged_attn_scratch(2, 1, hd), scale=1.0, lse=lse)
        o, l, mag, big = P.attend(_np(q), *c.seq(0), 1.0, 0)
        ds = 2.0 ** -19 * big + 1e-6
        u = P.U["bf16"]
        assert (np.abs(_np(out) - o) <= u * np.abs(o) + (u + 2 * ds[..., None]) * mag * 1.02 + 1e-7).all()
        assert (np.abs(_np(lse) - l) <= ds + 1e-6 * (1 + np.abs(l))).all()


def test_attn_many_sequences_of_many_rows(torch, m27b):
    rng = random.Random(41)
    q = [rng.choice([0, 2, 3, 4]) for _ in range(500)]
    _check_attn(torch, m27b, q, [x + rng.randrange(0, 40) for x in q], 128, 1, 128, "f16", 16, seed=42)


def test_attn_many_rows_same_every_time_other_stream_graph(torch, m27b):
    c = Cache(torch, m27b, [1500, 260], 16, 2, 256, "bf16", 43)
    q = torch.randn(560, 8, 256, device="cuda").bfloat16()
    cu, scr = _cu(torch, [300, 260]), m27b.paged_attn_scratch(8, 2, 256)
    want, out = torch.empty_like(q), torch.empty_like(q)
    m27b.paged_attn(c.kv, q, cu, c.lens, want, scr)
    for _ in range(8):
        m27b.paged_attn(c.kv, q, cu, c.lens, out, scr)
        assert torch.equal(out, want)
    torch.cuda.synchronize()
    out.zero_()
    s = torch.cuda.Stream()
    m27b.paged_attn(c.kv, q, cu, c.lens, out, scr, stream=s)
    s.synchronize()
    assert torch.equal(out, want)
    out.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m27b.paged_attn(c.kv, q, cu, c.lens, out, scr)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_attn_pages_before_the_window_may_be_gone(torch, m27b):
    # pages that no row sees: given back (-1) or anything
    for hd, nq, n_q, n_kv in ((128, 1, 16, 8), (256, 3, 8, 2), (128, 150, 8, 2), (256, 150, 8, 2)):
        n, ps, window = 900, 16, 100
        c = Cache(torch, m27b, [n], ps, n_kv, hd, "bf16", 44)
        first = (n - nq - window + 1) // ps  # the first page of the first row's window
        tab = c.table.clone()
        tab[0, :first] = -1
        tab[0, 0] = 1 << 30
        q = torch.randn(nq, n_q, hd, device="cuda").bfloat16()
        out = torch.empty_like(q)
        k, v = c.seq(0)
        page = c.tab[0, first]  # slots of the window's first page that no row sees
        gone = n - nq - window + 1 - first * ps
        if gone > 0:
            c.k[int(page), :gone], c.v[int(page), :gone] = float("inf"), float("nan")
        m27b.paged_attn(m27b.PagedKV(c.k, c.v, tab), q, _cu(torch, [nq]), c.lens, out, m27b.paged_attn_scratch(n_q, n_kv, hd), window=window)
        o, _, mag, _ = P.attend(_np(q), k, v, hd ** -0.5, window)
        assert (np.abs(_np(out) - o) <= 2.0 ** -8 * (np.abs(o) + 1.1 * mag) + 1e-6).all()
        assert m27b.device_status() == 0


def test_attn_token_offsets_are_held_to_the_buffers(torch, m27b):
    # offsets past the last token: what is there is attended, nothing beyond is touched
    c = Cache(torch, m27b, [50, 60], 16, 2, 64, "bf16", 45)
    q = torch.randn(4, 4, 64, device="cuda").bfloat16()
    wide = torch.full((6, 4, 64), 3.0, device="cuda").bfloat16()
    cu = torch.tensor([0, 2, 9], dtype=torch.int32, device="cuda")
    m27b.paged_attn(c.kv, q, cu, c.lens, wide[:4], m27b.paged_attn_scratch(4, 2, 64))
    o, _, mag, _ = P.attend(_np(q)[:2], *c.seq(0), 0.125, 0)
    assert (np.abs(_np(wide)[:2] - o) <= 2.0 ** -8 * (np.abs(o) + 1.1 * mag) + 1e-6).all()
    assert (wide[4:] == 3.0).all() and torch.isfinite(wide.float()).all()
    cu = torch.tensor([3, 1, 2], dtype=torch.int32, device="cuda")  # descending: no tokens
    wide.fill_(3.0)
    m27b.paged_attn(c.kv, q, cu, c.lens, wide[:4], m27b.paged_attn_scratch(4, 2, 64))
    assert (wide[[0, 2, 3]] == 3.0).all()


@pytest.mark.parametrize("hd,nq", [(64, 3), (128, 3), (128, 140)])
def test_attn_offsets_past_32_bits(torch, m27b, hd, nq):
    # pages 2^27 values apart: 40 of them reach past 2^32 values
    stride, ps, n_kv, n = 1 << 27, 16, 2, 37 * 16 + 5
    k = torch.empty(39 * stride + ps * n_kv * hd, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    kp, vp = (x.as_strided((40, ps, n_kv, hd), (stride, n_kv * hd, hd, 1)) for x in (k, v))
    for p in range(40):
        kp[p].normal_()
        vp[p].normal_()
    table = torch.arange(39, 0, -1, dtype=torch.int32, device="cuda").view(1, -1).contiguous()
    kv = m27b.PagedKV(kp, vp, table)
    q = torch.randn(nq, 4, hd, device="cuda").half()
    out = torch.empty_like(q)
    m27b.paged_attn(kv, q, _cu(torch, [nq]), torch.tensor([n], dtype=torch.int32, device="cuda"), out,
                    m27b.paged_attn_scratch(4, n_kv, hd))
    ids = table[0, :38].long()
    o, _, mag, _ = P.attend(_np(q), *(_np(x[ids]).reshape(-1, n_kv, hd)[:n] for x in (kp, vp)), hd ** -0.5, 0)
    assert (np.abs(_np(out) - o) <= 2.0 ** -11 * (np.abs(o) + 1.1 * mag) + 1e-6).all()


def test_attn_bad_pages_are_reported(torch, m27b):
    c = Cache(torch, m27b, [100], 16, 2, 64, "bf16", 19)
    for bad in (-1, 1 << 20):
        tab = c.table.clone()
        tab[0, 2] = bad
        q = torch.randn(1, 4, 64, device="cuda").bfloat16()
        m27b.paged_attn(m27b.PagedKV(c.k, c.v, tab), q, _cu(torch, [1]), c.lens, torch.empty_like(q),
                        m27b.paged_attn_scratch(4, 2, 64))
        assert m27b.device_status() == 6
    # a length past the table's end is held to it
    lens = torch.tensor([1 << 30], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 4, 64, device="cuda").bfloat16()
    m27b.paged_attn(c.kv, q, _cu(torch, [1]), lens, torch.empty_like(q), m27b.paged_attn_scratch(4, 2, 64))
    assert m27b.device_status() == 6
    rows = torch.tensor([7], dtype=torch.int32, device="cuda")
    m27b.paged_attn(c.kv, q, _cu(torch, [1]), c.lens, torch.empty_like(q), m27b.paged_attn_scratch(4, 2, 64), rows=rows)
    assert m27b.device_status() == 6


# --------------------------------------------------------------------------
# rotary positions and append


def _check_rope(torch, m27b, q_lens, kv_lens, n_q, n_kv, hd, dtype, src, ps, n_rot, interleaved, norm, seed, pad=0,
                rows=None, positions=None, in_place=False, v_inf=False):
    c = Cache(torch, m27b, kv_lens, ps, n_kv, hd, dtype, seed, pad=pad, rows=rows, poison=False)
    before = _np(c.k), _np(c.v)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    total, heads = sum(q_lens), n_q + 2 * n_kv
    x = (3 * torch.randn(total, heads, hd, generator=g, device="cuda")).to(_dt(torch, src))
    w = [1 + 0.3 * torch.randn(hd, generator=g, device="cuda") if norm in (True, s) else None for s in "qk"]
    if v_inf:
        x[::7, n_q + n_kv:, ::5] = float("inf")
    xn = _np(x)
    z = P.rope_factors(max(kv_lens) + 50, n_rot, 1e4)
    tab = torch.from_numpy(np.stack([z.real, z.imag], -1).astype(np.float32)).cuda().contiguous()
    z = np.stack([_np(tab)[..., 0] + 1j * _np(tab)[..., 1]])[0]  # the table as stored
    q_out = x[:, :n_q] if in_place else torch.zeros(total, n_q, hd, dtype=c.k.dtype, device="cuda")
    m27b.rope_append(c.kv, x[:, :n_q], x[:, n_q:n_q + n_kv], x[:, n_q + n_kv:], _cu(torch, q_lens), c.lens, tab, q_out,
                     interleaved=interleaved, q_norm=w[0], k_norm=w[1], eps=1e-5, rows=c.rows_t,
                     positions=None if positions is None else torch.tensor(positions, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    wn = [None if t is None else _np(t) for t in w]
    want_k, want_v = before[0].copy(), before[1].copy()
    want_q, at = np.zeros((total, n_q, hd)), 0
    for b, n in enumerate(q_lens):
        for i in range(n):
            p = kv_lens[b] - n + i
            rp = p if positions is None else positions[at]
            page, slot = c.tab[c.rows[b], p // ps], p % ps
            want_q[at] = P.norm_rope(xn[at, :n_q], wn[0], 1e-5, z[rp], n_rot, interleaved)
            want_k[page, slot] = P.norm_rope(xn[at, n_q:n_q + n_kv], wn[1], 1e-5, z[rp], n_rot, interleaved)
            want_v[page, slot] = xn[at, n_q + n_kv:]
            at += 1
    u = P.U[dtype]
    for got, want in ((_np(q_out), want_q), (_np(c.k), want_k), (_np(c.v), want_v)):
        same = np.isnan(want) | np.isinf(want)
        assert np.array_equal(got[same], want[same], equal_nan=True)
        big = np.abs(np.where(same, 0, want)).max(-1, keepdims=True)
        with np.errstate(invalid="ignore"):
            assert (np.abs(got - want) <= u * np.abs(want) + 2e-6 * big + 1e-7)[~same].all()
    if pad:
        assert torch.isfinite(c.buf[0][:, -pad:].float()).all()
    assert m27b.device_status() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("src", ["f32", "same"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,n_rot", [(256, 64), (256, 256), (128, 128), (128, 32), (64, 16), (64, 48), (64, 64)])
def test_rope_append(torch, m27b, dtype, src, interleaved, hd, n_rot):
    _check_rope(torch, m27b, [1, 5, 0, 33], [1, 40, 9, 33], 6, 2, hd, dtype, dtype if src == "same" else src, 16, n_rot,
                interleaved, True, seed=20)


@pytest.mark.parametrize("ps", [16, 64, 256])
@pytest.mark.parametrize("n_q,n_kv", [(1, 1), (24, 4), (3, 3), (0, 2)])
def test_rope_append_heads_pages(torch, m27b, ps, n_q, n_kv):
    if n_q == 0:
        c = Cache(torch, m27b, [20], ps, n_kv, 64, "bf16", 21, poison=False)
        x = torch.randn(3, 2 * n_kv, 64, device="cuda")
        tab = m27b.rope_table(32, 64, 1e4)
        m27b.rope_append(c.kv, None, x[:, :n_kv], x[:, n_kv:], _cu(torch, [3]), c.lens, tab, None)
        pages = [c.tab[0, p // ps] for p in (17, 18, 19)]
        got = torch.stack([c.v[int(a), p % ps] for a, p in zip(pages, (17, 18, 19))])
        assert torch.equal(got, x[:, n_kv:].bfloat16())
        return
    _check_rope(torch, m27b, [70, 1, 2], [300, 17, 2], n_q, n_kv, 128, "bf16", "f32", ps, 64, False, False, seed=22)


def test_rope_append_rows_positions_strides_in_place(torch, m27b):
    _check_rope(torch, m27b, [2, 4], [30, 20], 4, 2, 128, "bf16", "bf16", 16, 128, False, True, seed=23, pad=32, rows=[3, 1],
                positions=[5, 0, 31, 7, 7, 64])
    _check_rope(torch, m27b, [9], [30], 4, 2, 256, "f16", "f16", 32, 64, True, True, seed=24, in_place=True)


def test_rope_append_many_sequences(torch, m27b):
    rng = random.Random(25)
    q = [rng.choice([0, 1, 2, 3]) for _ in range(1300)]
    _check_rope(torch, m27b, q, [x + rng.randrange(20) for x in q], 2, 1, 64, "bf16", "f32", 16, 64, False, False, seed=26)


@pytest.mark.parametrize("n_q,n_kv,hd,src,dtype,ps", [(2, 1, 64, "f32", "bf16", 16), (40, 8, 256, "f32", "bf16", 64),
                                                      (16, 8, 128, "f16", "f16", 32), (6, 2, 256, "bf16", "bf16", 128)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_append_many_tokens(torch, m27b, n_q, n_kv, hd, src, dtype, ps, interleaved):
    # enough tokens for the streaming kernel; 40 + 16 heads of 256 fp32 values are two units a token
    _check_rope(torch, m27b, [1200, 0, 700], [1200, 5, 1000], n_q, n_kv, hd, dtype, src, ps, hd // 2, interleaved, True, seed=50,
                rows=[2, 0, 1])


@pytest.mark.parametrize("n_q,n_kv,hd,n_rot,norm", [(3, 2, 64, 16, "q"), (5, 1, 64, 48, "k"), (5, 3, 128, 32, "k"),
                                                    (1, 1, 128, 16, True), (3, 2, 256, 16, "q"), (9, 5, 128, 128, True)])
def test_rope_append_many_tokens_mixed_heads(torch, m27b, n_q, n_kv, hd, n_rot, norm):
    # q, k and v heads in one warp, of which only some are normalised and turned
    _check_rope(torch, m27b, [640, 1, 9], [700, 1, 30], n_q, n_kv, hd, "bf16", "f32", 16, n_rot, False, norm, seed=53, v_inf=True)
    _check_rope(torch, m27b, [650], [651], n_q, n_kv, hd, "f16", "f16", 64, n_rot, True, norm, seed=54, v_inf=True)


def test_rope_append_many_tokens_in_place_and_left_out(torch, m27b):
    _check_rope(torch, m27b, [1900], [2000], 4, 2, 128, "f16", "f16", 32, 64, True, False, seed=51, in_place=True)
    # tokens of no sequence, and positions past the table, among many
    c = Cache(torch, m27b, [1000], 16, 1, 64, "bf16", 52, poison=False)
    x = torch.randn(3000, 3, 64, device="cuda")
    q = torch.full((3000, 1, 64), 9.0, device="cuda").bfloat16()
    k0 = c.k.clone()
    m27b.rope_append(c.kv, x[:, :1], x[:, 1:2], x[:, 2:], torch.tensor([100, 1100], dtype=torch.int32, device="cuda"), c.lens,
                     m27b.rope_table(990, 64, 1e4), q)
    assert m27b.device_status() == 6
    assert (q[:100] == 9.0).all() and (q[1090:] == 9.0).all() and not (q[100:1090] == 9.0).all(-1).any()
    page = int(c.tab[0, 62])  # positions 992..: past the table
    assert torch.equal(c.k[page], k0[page])
    assert m27b.device_status() == 0


def test_rope_append_out_of_range_is_left_out(torch, m27b):
    c = Cache(torch, m27b, [20], 16, 1, 64, "bf16", 27, poison=False)
    k0 = c.k.clone()
    x = torch.randn(3, 3, 64, device="cuda")
    tab = m27b.rope_table(19, 64, 1e4)  # position 19 has no entry
    q = torch.zeros(3, 1, 64, dtype=torch.bfloat16, device="cuda")
    m27b.rope_append(c.kv, x[:, :1], x[:, 1:2], x[:, 2:], _cu(torch, [3]), c.lens, tab, q)
    assert m27b.device_status() == 6
    assert (q[2] == 0).all() and (q[:2] != 0).any()
    page = int(c.tab[0, 1])
    assert torch.equal(c.k[page, 3].nan_to_num(), k0[page, 3].nan_to_num())  # position 19
    assert not torch.equal(c.k[page, 2], k0[page, 2])
    for tab2, ln in (([5, -1], 20), ([5, 1 << 29], 20), ([5, 1], 1), ([5, 1], 5000)):
        t = torch.tensor([tab2], dtype=torch.int32, device="cuda").clamp(max=1 << 29)
        t[0, 0] = min(5, c.k.shape[0] - 1)
        k1 = c.k.clone()
        kv = m27b.PagedKV(c.k, c.v, t)
        m27b.rope_append(kv, x[:, :1], x[:, 1:2], x[:, 2:], _cu(torch, [3]),
                         torch.tensor([ln], dtype=torch.int32, device="cuda"), m27b.rope_table(6000, 64, 1e4), q)
        assert m27b.device_status() == 6
        if ln != 1:
            assert torch.equal(c.k.nan_to_num(), k1.nan_to_num())
        c.k.copy_(k1)


@pytest.mark.parametrize("kind", ["none", "linear", "yarn"])
@pytest.mark.parametrize("n_rot,theta", [(64, 1e7), (128, 1e4), (2, 10.0)])
def test_rope_table(torch, m27b, kind, n_rot, theta):
    n = 200001
    code = {"none": m27b.ROPE_NONE, "linear": m27b.ROPE_LINEAR, "yarn": m27b.ROPE_YARN}[kind]
    got = _np(m27b.rope_table(n, n_rot, theta, kind=code, factor=1.0 if kind == "none" else 8.0, original_ctx=4096))
    z = P.rope_factors(n, n_rot, theta, kind, 8.0, 4096)
    # one fp32 rounding of values up to 1.3, and an angle up to 2e5 off by 2^-52 of it in fp64
    assert np.abs(got[..., 0] - z.real).max() <= 2.0 ** -23 and np.abs(got[..., 1] - z.imag).max() <= 2.0 ** -23


# --------------------------------------------------------------------------
# pages


class Upkeep:
    """A PageSet beside its plain restatement."""

    def __init__(self, torch, m27b, n_rows, n_cols, n_pages, ps, planes=3, width=24, pools=1, seed=0):
        self.torch, self.m = torch, m27b
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.pool = [torch.randn(planes, n_pages, width, generator=g, device="cuda") for _ in range(pools)]
        self.ps = m27b.PageSet.empty(n_rows, n_cols, n_pages, ps, self.pool)
        self.ref = P.Pages(n_rows, n_cols, n_pages, ps, [list(pl) for p in self.pool for pl in p.cpu().numpy().copy()])

    def i(self, v):
        return self.torch.tensor(v, dtype=self.torch.int32, device="cuda")

    def do(self, op, *lists):
        want = getattr(self.ref, op)(*lists)
        getattr(self.ps, op)(*(self.i(v) for v in lists))
        self.same()
        if want in ("bad", "full"):
            with pytest.raises(self.m.M27BError, match="too few" if want == "full" else "bad request"):
                self.ps.check()
        else:
            self.ps.check()
        return want

    def same(self):
        assert self.ps.table.tolist() == self.ref.table
        assert self.ps.ref.tolist() == self.ref.ref
        assert self.ps.lens.tolist() == self.ref.lens
        got = np.concatenate([p.cpu().numpy() for p in self.pool])
        assert np.array_equal(got, np.array(self.ref.data))
        assert self.m.device_status() == 0


@pytest.mark.parametrize("ps", [1, 16, 64])
@pytest.mark.parametrize("pools,width", [(1, 4), (2, 24), (1, 20000)])
def test_pages_random_life(torch, m27b, ps, pools, width):
    rng = random.Random(ps * 100 + pools)
    n_rows, n_cols, n_pages = 12, 9, 40
    u = Upkeep(torch, m27b, n_rows, n_cols, n_pages, ps, width=width, pools=pools)
    seen = set()
    for _ in range(60):
        op = rng.choice(["resize", "resize", "resize", "fork", "fork", "free", "compact"])
        if op == "resize":
            rows = rng.sample(range(n_rows), rng.randint(1, 4))
            seen.add(u.do("resize", rows, [rng.randint(0, n_cols * ps) for _ in rows]))
        elif op == "fork":
            empty = [r for r in range(n_rows) if u.ref.lens[r] == 0]
            full = [r for r in range(n_rows) if u.ref.lens[r] > 0]
            if not empty or not full:
                continue
            dst = rng.sample(empty, rng.randint(1, len(empty)))
            seen.add(u.do("fork", [rng.choice(full) for _ in dst], dst))
        elif op == "free":
            rows = rng.sample(range(n_rows), rng.randint(1, 5))
            u.ref.free(rows)
            u.ps.free(u.i(rows))
            u.same()
        else:
            live = u.i([0])
            want = u.ref.compact()
            u.ps.compact(n_live=live)
            u.same()
            assert int(live) == want
    assert None in seen


def test_pages_refusals_change_nothing(torch, m27b):
    u = Upkeep(torch, m27b, 6, 4, 8, 16)
    assert u.do("resize", [0, 1], [50, 17]) is None
    assert u.do("resize", [2], [64]) == "full"  # 2 of 4 pages are left
    assert u.do("resize", [2, 2], [1, 2]) == "bad"
    assert u.do("resize", [2], [65]) == "bad"
    assert u.do("resize", [2], [-1]) == "bad"
    assert u.do("resize", [6], [1]) == "bad"
    assert u.do("resize", [2, -1], [1, 1]) == "bad"
    assert u.do("fork", [0, 0, 0], [2, 3, 4]) == "full"
    assert u.do("fork", [0], [1]) == "bad"
    assert u.do("fork", [0, 0], [2, 2]) == "bad"
    assert u.do("fork", [0, 2], [2, 3]) == "bad"
    assert u.do("fork", [0], [9]) == "bad"
    assert u.do("fork", [-2], [2]) == "bad"
    assert u.do("fork", [0, 1], [2, 3]) is None


def test_pages_shared_half_page_is_copied_before_it_grows(torch, m27b):
    u = Upkeep(torch, m27b, 5, 4, 20, 16)
    u.do("resize", [0], [64])
    u.do("fork", [0, 0], [1, 2])      # whole pages only: shared, no copy
    u.do("resize", [1, 2], [40, 41])  # back into the middle of a shared page
    u.do("resize", [1, 2, 0], [44, 41, 64])
    u.do("resize", [0, 2], [33, 64])
    u.do("resize", [0], [40])
    assert u.ref.table[1][2] != u.ref.table[2][2] != u.ref.table[0][2]


def test_pages_free_twice_and_many(torch, m27b):
    u = Upkeep(torch, m27b, 2000, 6, 9000, 4, planes=1, width=4)
    rng = random.Random(5)
    rows = list(range(1500))
    u.do("resize", rows, [rng.randint(0, 20) for _ in rows])
    u.do("fork", [rng.choice(rows) for _ in range(500)], list(range(1500, 2000)))
    gone = rng.sample(range(2000), 900)
    u.ref.free(gone)
    u.ps.free(u.i(gone + gone[:300]))
    u.same()
    u.ref.compact()
    u.ps.compact()
    u.same()
    u.ps.compact()
    u.same()


def test_pages_copy_and_strided_pools(torch, m27b):
    base = torch.randn(4, 30, 2, 16, device="cuda").bfloat16()  # keys and values of a page side by side
    k, v = base[:, :, 0], base[:, :, 1]
    want = base.clone()
    ps = m27b.PageSet.empty(3, 3, 30, 16, [k, v])
    src, dst = [3, 4, 3, 29], [0, 1, 2, 5]
    want[:, dst] = want[:, src]
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    ps.copy(i(src), i(dst))
    assert torch.equal(base, want) and m27b.device_status() == 0
    ps.copy(i([3, 30]), i([-1, 2]))
    assert torch.equal(base, want) and m27b.device_status() == 6


def test_pages_graph(torch, m27b):
    u = Upkeep(torch, m27b, 6, 4, 30, 16)
    u.do("resize", [0, 1], [50, 33])
    src, dst = u.i([0, 1]), u.i([2, 3])
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        u.ps.fork(src, dst)
        u.ps.free(dst)
        u.ps.fork(src, dst)
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        u.ref.free([2, 3])
        assert u.ref.fork([0, 1], [2, 3]) is None
        if _ == 0:
            u.same()
            u.ps.free(dst)
            u.ref.free([2, 3])
    u.same()


# --------------------------------------------------------------------------
# all of it together


def test_example_runs(torch, m27b, capsys):
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_serving.py")
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    ex.main()
    assert "pages in use" in capsys.readouterr().out


def test_forked_sequences_go_on_apart(torch, m27b):
    # a fork, then different tokens: each row's cache is its own from there on,
    # and equals one built without a fork
    ps, n_kv, hd = 16, 2, 64
    pool = torch.randn(2, 60, ps, n_kv, hd, device="cuda").bfloat16()
    pages = m27b.PageSet.empty(4, 10, 60, ps, pool)
    kv = m27b.PagedKV(pool[0], pool[1], pages.table)
    rope, scr = m27b.rope_table(200, hd, 1e4), m27b.paged_attn_scratch(4, n_kv, hd)
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731

    def add(row, x):
        n = len(x)
        pages.resize(i(row), pages.lens[row:row + 1] + n)
        q, o = (torch.empty(n, 4, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        m27b.rope_append(kv, x[:, :4], x[:, 4:6], x[:, 6:], i(0, n), pages.lens, rope, q, rows=i(row))
        m27b.paged_attn(kv, q, i(0, n), pages.lens, o, scr, rows=i(row))
        return o

    x = [torch.randn(n, 8, hd, device="cuda") for n in (37, 5, 30, 1)]
    add(0, x[0])
    pages.fork(i(0), i(1))
    left, right = add(0, x[1]), add(1, x[2])
    right2 = add(1, x[3])
    add(2, x[0])
    assert torch.equal(add(2, x[1]), left)
    pages.free(i(0, 2))
    pages.compact()
    add(3, x[0])
    assert torch.equal(add(3, x[2]), right) and torch.equal(add(3, x[3]), right2)
    pages.check()
    assert int((pages.ref > 0).sum()) == 2 * P.cdiv(68, ps)
