"""Edges of the paged attention on the GPU (include/m27b_paged.h) against a
plain 64-bit computation.

Tolerances: those of tests/test_paged_gpu.py (u: half a unit in the last place,
relative; ds: the scores' fp32 sums).  A weight below f16's 2^-14 has an error of
at most 2^-25 absolute; the largest weight is at least 2^7, so that adds at most
2^-32 sum |v| for f16."""
import random

import numpy as np
import pytest

import _paged_ref as P
from test_paged_gpu import Cache, _cu

pytestmark = pytest.mark.gpu


def _attend(torch, q, k, v, scale, window):
    """One sequence: out, lse, sum p |v|, the row's largest scale * sum |q| |k|, and sum |v|."""
    nq, n_q, hd = q.shape
    nkv, n_kv = k.shape[:2]
    q, k, v = q.double(), k.double().repeat_interleave(n_q // n_kv, 1), v.double().repeat_interleave(n_q // n_kv, 1)
    hi = torch.arange(nq, device="cuda") + nkv - nq + 1
    pos = torch.arange(nkv, device="cuda")
    see = pos < hi[:, None]
    if window > 0:
        see &= pos >= hi[:, None] - window
    see = see[:, None]
    s = (scale * torch.einsum("thd,xhd->thx", q, k)).masked_fill(~see, -np.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.masked_fill(lse == -np.inf, 0.0)[..., None])
    big = (scale * torch.einsum("thd,xhd->thx", q.abs(), k.abs())).masked_fill(~see, 0.0)
    big = big.amax(-1) if nkv else lse.masked_fill(lse == -np.inf, 0.0)
    some = torch.einsum("thx,xhd->thd", see.expand_as(s).double(), v.abs())
    return torch.einsum("thx,xhd->thd", p, v), lse, torch.einsum("thx,xhd->thd", p, v.abs()), big, some


def _close(torch, got, lse, want, dtype):
    out, l, mag, big, some = want
    ds, u = 2.0 ** -19 * big + 1e-6, P.U[dtype]
    tol = u * out.abs() + (u + 2 * ds[..., None]) * mag * 1.02 + 1e-7
    if dtype == "f16":
        tol = tol + 2.0 ** -32 * some
    err = (got.double() - out).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    if lse is not None:
        f = torch.isfinite(l)
        assert torch.equal(lse == -np.inf, l == -np.inf)
        assert bool(((lse.double() - l).abs() <= ds + 1e-6 * (1 + l.abs()))[f].all())


def _seq(torch, c, b):
    n = c.lens_list[b]
    ids = c.table[c.rows[b], :P.cdiv(n, c.ps)].long()
    return tuple(x[ids].reshape(-1, *x.shape[2:])[:n] for x in (c.k, c.v))


def _run(torch, m27b, c, q, cu, **kw):
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    m27b.paged_attn(c.kv, q, cu, c.lens, out, m27b.paged_attn_scratch(q.shape[1], c.kv.n_kv, q.shape[2]), lse=lse,
                    rows=c.rows_t, **kw)
    return out, lse


@pytest.mark.parametrize("hd,dtype,n_q,n_kv", [(128, "f16", 16, 8), (128, "bf16", 12, 2), (256, "bf16", 12, 2)])
def test_items_of_one_two_and_three_tiles_with_idle_quarters(torch, m27b, hd, dtype, n_q, n_kv):
    # many prompts whose row tiles see one key tile, two and three, the last ones
    # with idle warps or an idle second CTA, so that a pair has such items in a row
    rng = random.Random(50)
    per = 2 * (128 // (n_q // n_kv))  # tokens of a pair's item
    q_lens = [rng.choice([per, 2 * per + 1, 2 * per + per // 3, 3 * per, per + 5, 3 * per + 1]) for _ in range(70)]
    if per < 128:  # key tiles of 128 positions
        kv = [n + rng.choice([0, 0, 128 - per, 256 - per, 300]) for n in q_lens]
    else:
        kv = list(q_lens)
    c = Cache(torch, m27b, kv, 16, n_kv, hd, dtype, 51)
    q = torch.randn(sum(q_lens), n_q, hd, device="cuda").to(c.k.dtype)
    cu = _cu(torch, q_lens)
    out, lse = _run(torch, m27b, c, q, cu)
    at = 0
    for b, n in enumerate(q_lens):
        if b % 7 == 0:
            _close(torch, out[at:at + n], lse[at:at + n], _attend(torch, q[at:at + n], *_seq(torch, c, b), hd ** -0.5, 0), dtype)
        at += n
    for _ in range(200):
        again, lse2 = _run(torch, m27b, c, q, cu)
        assert torch.equal(again, out) and torch.equal(lse2, lse)
    assert m27b.device_status() == 0


@pytest.mark.parametrize("hd,q_lens,kv_lens", [(64, [13, 1, 40], [3, 90, 20]), (128, [13, 1], [3, 90]), (128, [300, 90], [100, 70]),
                                               (256, [300, 150], [290, 150])])
def test_a_window_of_any_size(torch, m27b, hd, q_lens, kv_lens):
    # a window that reaches past the cache is none, up to the type's end, also
    # where a sequence has fewer positions than new tokens
    c = Cache(torch, m27b, kv_lens, 16, 2, hd, "bf16", 52)
    q = torch.randn(sum(q_lens), 8, hd, device="cuda").bfloat16()
    cu = _cu(torch, q_lens)
    want = _run(torch, m27b, c, q, cu)
    at = 0
    for b, n in enumerate(q_lens):
        _close(torch, want[0][at:at + n], want[1][at:at + n], _attend(torch, q[at:at + n], *_seq(torch, c, b), hd ** -0.5, 0), "bf16")
        at += n
    for window in (2 ** 31 - 1, 2 ** 31 - 200, 2 ** 30, c.tab.shape[1] * 16, -1):
        got = _run(torch, m27b, c, q, cu, window=window)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), window
    assert m27b.device_status() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd,q_lens,kv_lens", [
    (64, [1, 3, 40], [500, 3, 41]),           # whole items
    (256, [1, 1], [9000, 40]),                # an item over many workers, joined
    (128, [300, 150], [300, 150]),            # pairs
    (128, [100], [6000]), (256, [140], [4000]),  # pairs, joined
])
def test_a_nan_in_q_stays_one(torch, m27b, dtype, hd, q_lens, kv_lens):
    # a row whose scores are NaN is NaN, not the zeros of a row that sees nothing;
    # the other rows are as without it
    c = Cache(torch, m27b, kv_lens, 16, 2, hd, dtype, 53)
    q = torch.randn(sum(q_lens), 4, hd, device="cuda").to(c.k.dtype)
    cu = _cu(torch, q_lens)
    out, lse = _run(torch, m27b, c, q, cu)
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[-1, 2] = bad[len(q) // 2, 0] = True
    q[bad.nonzero()[:, 0], bad.nonzero()[:, 1], hd // 3] = float("nan")
    got, got_l = _run(torch, m27b, c, q, cu)
    assert bool(torch.isnan(got[bad]).all()) and bool(torch.isnan(got_l[bad]).all())
    assert torch.equal(got[~bad], out[~bad]) and torch.equal(got_l[~bad], lse[~bad])
    assert m27b.device_status() == 0


@pytest.mark.parametrize("hd,kv_len", [(64, 700), (128, 9000)])
def test_a_nan_key_that_a_row_sees_is_not_an_empty_row(torch, m27b, hd, kv_len):
    c = Cache(torch, m27b, [kv_len, 200], 16, 2, hd, "bf16", 54)
    q = torch.randn(2, 4, hd, device="cuda").bfloat16()
    cu = _cu(torch, [1, 1])
    out, lse = _run(torch, m27b, c, q, cu)
    c.k[int(c.tab[0, 10]), 3, 1, 5] = float("nan")  # kv head 1: query heads 2 and 3
    got, got_l = _run(torch, m27b, c, q, cu)
    assert bool(torch.isnan(got[0, 2:]).all()) and bool(torch.isnan(got_l[0, 2:]).all())
    assert torch.equal(got[0, :2], out[0, :2]) and torch.equal(got[1], out[1]) and torch.equal(got_l[1], lse[1])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd,n_seq,n_tok,group", [(64, 200, 1, 1), (128, 200, 1, 2), (256, 200, 1, 2), (128, 90, 12, 16), (256, 90, 12, 16)])
@pytest.mark.parametrize("sink", ["first", "last"])
def test_many_small_weights_beside_a_large_one(torch, m27b, dtype, hd, n_seq, n_tok, group, sink):
    # one position with nearly all of the weight and a value of 0, and 40000 whose
    # weights are 2^-25.25 to 2^-26 of its: the result is what these add up to.  All rows of the
    # table hold the same pages; with so many sequences no worker has less than
    # about half of one.
    n, ps = 40000, 64
    g = torch.Generator(device="cuda").manual_seed(55)
    c = Cache(torch, m27b, [n], ps, 1, hd, dtype, 56)
    d = torch.randint(25 * 8 + 2, 26 * 8 + 1, (n,), generator=g, device="cuda") / 8  # exact in both types
    key, val = torch.zeros(n, 1, hd, device="cuda"), 0.5 + torch.rand(n, 1, hd, generator=g, device="cuda")
    at = 0 if sink == "first" else n - n_tok
    d[at] = 0
    key[:, 0, 0], val[at] = -d, 0.0
    ids = c.table[0, :P.cdiv(n, ps)].long()
    c.k[ids], c.v[ids] = key.to(c.k.dtype).view(-1, ps, 1, hd), val.to(c.v.dtype).view(-1, ps, 1, hd)
    q = torch.zeros(n_seq * n_tok, group, hd, device="cuda", dtype=c.k.dtype)
    q[..., 0] = 1.0
    kv = m27b.PagedKV(c.k, c.v, c.table.repeat(n_seq, 1).contiguous())
    lens, scale = torch.full((n_seq,), n, dtype=torch.int32, device="cuda"), float(np.log(2.0))
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    m27b.paged_attn(kv, q, _cu(torch, [n_tok] * n_seq), lens, out, m27b.paged_attn_scratch(group, 1, hd), scale=scale, lse=lse)
    want = _attend(torch, q[:n_tok], *_seq(torch, c, 0), scale, 0)
    for b in range(0, n_seq, 13):
        _close(torch, out[b * n_tok:(b + 1) * n_tok], lse[b * n_tok:(b + 1) * n_tok], want, dtype)
    assert m27b.device_status() == 0


def test_rope_table_on_another_stream_takes_no_memory_in_use(torch, m27b):
    want = m27b.rope_table(20000, 128, 1e4)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(3):
        old = torch.empty_like(want)
        torch.cuda._sleep(20000000)
        old.fill_(7.0)  # runs after the sleep
        del old         # and its memory is free for this stream's next tensor
        got = m27b.rope_table(20000, 128, 1e4, stream=s)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("hd,q_lens,kv_lens", [(64, [1, 5, 1], [100, 90, 300]), (128, [150, 200, 90], [150, 300, 400])])
def test_a_bad_page_counts_as_zeros_in_its_own_sequence(torch, m27b, hd, q_lens, kv_lens):
    c = Cache(torch, m27b, kv_lens, 16, 2, hd, "bf16", 57)
    q = torch.randn(sum(q_lens), 8, hd, device="cuda").bfloat16()
    cu = _cu(torch, q_lens)
    out, lse = _run(torch, m27b, c, q, cu)
    k, v = _seq(torch, c, 1)
    k[32:48] = v[32:48] = 0.0
    mine = slice(q_lens[0], q_lens[0] + q_lens[1])
    want = _attend(torch, q[mine], k, v, hd ** -0.5, 0)
    for bad in (-1, c.k.shape[0], 1 << 30):
        c.table[1, 2] = bad
        got, got_l = _run(torch, m27b, c, q, cu)
        assert m27b.device_status() == 6
        _close(torch, got[mine], got_l[mine], want, "bf16")
        for o in (slice(0, mine.start), slice(mine.stop, None)):
            assert torch.equal(got[o], out[o]) and torch.equal(got_l[o], lse[o])
    # a length beyond the table, and a row beyond it
    c.table[1, 2] = int(c.tab[1, 2])
    lens = c.lens.clone()
    lens[1] = 1 << 30
    got = torch.full_like(q, 7.0)
    m27b.paged_attn(c.kv, q, cu, lens, got, m27b.paged_attn_scratch(8, 2, hd))
    assert m27b.device_status() == 6
    rows = torch.tensor([0, 3, 2], dtype=torch.int32, device="cuda")
    none = torch.full_like(q, 7.0)
    m27b.paged_attn(c.kv, q, cu, c.lens, none, m27b.paged_attn_scratch(8, 2, hd), rows=rows)
    assert m27b.device_status() == 6 and bool((none[mine] == 0).all())
    for b, o in ((0, slice(0, mine.start)), (2, slice(mine.stop, None))):  # the work is cut elsewhere: not bit for bit
        want = _attend(torch, q[o], *_seq(torch, c, b), hd ** -0.5, 0)
        _close(torch, got[o], None, want, "bf16")
        _close(torch, none[o], None, want, "bf16")


def test_steps_back_to_back_read_what_the_launch_before_wrote(torch, m27b):
    # resize, append, attention of 70 rows, five steps in one graph, where each
    # launch begins before the one before it has ended; and with a wait after each
    ps, n_kv, hd, n_q, n = 16, 2, 128, 8, 70
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    rope, scr = m27b.rope_table(400, hd, 1e4), m27b.paged_attn_scratch(n_q, n_kv, hd)
    rows, cu = i(list(range(n))), i(list(range(n + 1)))
    x = torch.randn(5, n, n_q + 2 * n_kv, hd, device="cuda")
    results = []
    for graphed in (False, True):
        pool = torch.zeros(2, 1000, ps, n_kv, hd, device="cuda").bfloat16()
        pages = m27b.PageSet.empty(n, 20, 1000, ps, pool)
        kv = m27b.PagedKV(pool[0], pool[1], pages.table)
        start = i([(7 * r) % 150 for r in range(n)])
        pages.resize(rows, start)
        lens = [start + 1 + s for s in range(5)]
        q, out = (torch.zeros(5, n, n_q, hd, device="cuda").bfloat16() for _ in range(2))
        wait = (lambda: None) if graphed else torch.cuda.synchronize

        def steps():
            for s in range(5):
                pages.resize(rows, lens[s])
                wait()
                m27b.rope_append(kv, x[s, :, :n_q], x[s, :, n_q:n_q + n_kv], x[s, :, n_q + n_kv:], cu, pages.lens, rope, q[s])
                wait()
                m27b.paged_attn(kv, q[s], cu, pages.lens, out[s], scr)
                wait()

        torch.cuda.synchronize()
        if graphed:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                steps()
            for _ in range(20):
                pages.resize(rows, start)
                pool.zero_()
                out.zero_()
                g.replay()
                pages.check()
                results.append((out.clone(), pages.lens.clone()))
        else:
            steps()
            pages.check()
            results.append((out.clone(), pages.lens.clone()))
    for o, ln in results[1:]:
        assert torch.equal(o, results[0][0]) and torch.equal(ln, results[0][1])
    assert m27b.device_status() == 0
