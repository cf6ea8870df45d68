"""Performance cases of the paged key/value cache: rotary positions with the
append to the cache, attention of new tokens over it, and the upkeep of its
pages.

A case names an operator ("rope_append", "attend", "fork" or "turnover") and
its sizes; the lengths of a batch's sequences are drawn from the case's own
`shape` number, the values from the seed.  `run` computes the operators with
elementary torch operations in 32 bits, or, where `own` is true, through the
package's public entry points.  `exact` restates each definition in 64 bits,
sequence by sequence.

The cache: one layer's pools hold element d of kv head j at slot s of page p
at k[p, s, j, d]; position i of the sequence in table row r lives in page
table[r, i // page] at slot i % page.  New tokens of sequence b are rows
cu_q[b] .. cu_q[b + 1] of q, the last of them at position lens[b] - 1.
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _m27b():
    pkg = os.path.join(_ROOT, "mono-qwen27_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import m27b
    return m27b


# --------------------------------------------------------------------------
# cases


def listed():
    big = dict(n_q=24, n_kv=4, hd=256)    # the repository's 64-layer model
    small = dict(n_q=16, n_kv=8, hd=128)  # its 28-layer draft
    return [
        # one user's next token, a short conversation: latency
        dict(name="attend: a token, short", op="attend", n_seq=1, q_lo=1, q_hi=1, kv_lo=769, kv_hi=769, dtype="bf16",
             page=16, window=0, lse=False, odd=False, shape=1, **big),
        # a full decode batch of ragged conversations: the cache is read once
        dict(name="attend: decode batch", op="attend", n_seq=64, q_lo=1, q_hi=1, kv_lo=300, kv_hi=8192, dtype="bf16",
             page=64, window=0, lse=False, odd=False, shape=2, **big),
        # one long document, a token at a time: the split over positions
        dict(name="attend: a token, long", op="attend", n_seq=1, q_lo=1, q_hi=1, kv_lo=131071, kv_hi=131071,
             dtype="f16", page=32, window=0, lse=True, odd=False, shape=3, **small),
        # drafted tokens of eight sequences under verification
        dict(name="attend: verify", op="attend", n_seq=8, q_lo=8, q_hi=8, kv_lo=1000, kv_hi=6000, dtype="bf16", page=16,
             window=0, lse=False, odd=False, shape=4, **big),
        # a batch of prompts of many lengths, some idle or empty, sliding window
        dict(name="attend: ragged prompts", op="attend", n_seq=7, q_lo=1, q_hi=2047, kv_lo=33, kv_hi=4095, dtype="f16",
             page=16, window=1500, lse=True, odd=True, shape=5, **small),
        # the second half of a long prompt: matrix products
        dict(name="attend: prompt chunk", op="attend", n_seq=1, q_lo=4096, q_hi=4096, kv_lo=8192, kv_hi=8192,
             dtype="bf16", page=64, window=0, lse=False, odd=False, shape=6, **big),
        # one user's next token: head norms, rotation and append of fp32 projections
        dict(name="rope: a token", op="rope_append", n_seq=1, q_lo=1, q_hi=1, kv_lo=769, kv_hi=769, dtype="bf16",
             src="f32", page=16, n_rot=64, interleaved=False, norm=True, scaling="none", shape=7, **big),
        # a decode batch in 16 bits, whole heads in interleaved pairs, stretched positions
        dict(name="rope: decode batch", op="rope_append", n_seq=64, q_lo=1, q_hi=1, kv_lo=300, kv_hi=60000, dtype="f16",
             src="f16", page=32, n_rot=128, interleaved=True, norm=False, scaling="yarn", shape=8, **small),
        # prompts: a pass over the projections
        dict(name="rope: prompts", op="rope_append", n_seq=3, q_lo=1500, q_hi=4095, kv_lo=1500, kv_hi=20001,
             dtype="bf16", src="f32", page=64, n_rot=64, interleaved=False, norm=True, scaling="linear", shape=9, **big),
        # one prompt answered four ways, and the answers dropped again
        dict(name="pages: four answers", op="fork", n_seq=3, n_child=4, len_lo=200, len_hi=900, page=16, planes=56,
             page_bytes=32768, spare=9, shape=10),
        # many beams: page tables, counts and the copies of half-filled pages
        dict(name="pages: many beams", op="fork", n_seq=24, n_child=120, len_lo=100, len_hi=6000, page=16, planes=56,
             page_bytes=32768, spare=100, shape=11),
        # half of the sequences end and the pages that are left move together
        dict(name="pages: turnover", op="turnover", n_seq=48, n_child=0, len_lo=50, len_hi=900, page=16, planes=56,
             page_bytes=32768, spare=150, shape=12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "rope_append", "rope_append", "fork", "turnover"])
    shape = rng.randrange(1 << 30)
    if op in ("fork", "turnover"):
        page = rng.choice([16, 32, 64])
        n_seq = _log_int(rng, 2, 40)
        page_bytes = page * rng.choice([512, 1024, 2048])
        return dict(op=op, n_seq=n_seq, n_child=_log_int(rng, 1, 100) if op == "fork" else 0, len_lo=rng.randint(1, 100),
                    len_hi=_log_int(rng, 101, 600), page=page, planes=2 * rng.randint(1, 28 * 32768 // max(page_bytes, 32768)),
                    page_bytes=page_bytes, spare=rng.randint(0, 150), shape=shape)
    n_kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 6, 8])
    hd = rng.choice([64, 128, 256])
    n_q = n_kv * group
    dtype = rng.choice(["bf16", "f16"])
    page = rng.choice([16, 32, 64, 128])
    if op == "rope_append":
        n_seq = _log_int(rng, 1, 64)
        q_hi = _log_int(rng, 1, max(1, 9000 // n_seq))
        kv_hi = _log_int(rng, q_hi + 1, 60000)
        return dict(op=op, n_seq=n_seq, q_lo=rng.randint(1, q_hi), q_hi=q_hi, kv_lo=q_hi, kv_hi=kv_hi, n_q=n_q,
                    n_kv=n_kv, hd=hd, dtype=dtype, src=rng.choice(["f32", dtype]), page=page,
                    n_rot=rng.choice([hd // 4, hd // 2, hd]), interleaved=rng.random() < 0.5, norm=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "yarn"]), shape=shape)
    kind = rng.choice(["decode", "verify", "prompt"])
    if kind == "decode":
        n_seq, q_lo, q_hi = _log_int(rng, 1, 64), 1, 1
        kv_hi = _log_int(rng, 17, max(18, min(300000, 150000000 // (n_kv * hd)) // n_seq))
    elif kind == "verify":
        n_seq, q_lo, q_hi = _log_int(rng, 1, 16), rng.randint(1, 4), rng.randint(5, 16)
        kv_hi = _log_int(rng, 17, 8000)
    else:
        n_seq = rng.randint(1, 6)
        q_lo, q_hi = rng.randint(1, 100), _log_int(rng, 101, 2000)
        kv_hi = _log_int(rng, q_hi, 4500)
    return dict(op=op, n_seq=n_seq, q_lo=q_lo, q_hi=q_hi, kv_lo=_log_int(rng, 1, kv_hi), kv_hi=kv_hi, n_q=n_q, n_kv=n_kv,
                hd=hd, dtype=dtype, page=page, window=rng.choice([0, 0, 0, _log_int(rng, 1, 2000)]),
                lse=rng.random() < 0.5, odd=rng.random() < 0.5, shape=shape)


def _lengths(case):
    """New tokens and cached positions (the new ones among them) of each sequence."""
    rng = random.Random(case["shape"])
    q, kv = [], []
    for b in range(case["n_seq"]):
        nq = _log_int(rng, case["q_lo"], case["q_hi"])
        nkv = max(nq, _log_int(rng, case["kv_lo"], case["kv_hi"]))
        if case.get("odd") and b == 1:
            nq = 0  # an idle sequence
        if case.get("odd") and b == 2:
            nkv = 0  # nothing cached: every row is empty
        if case.get("odd") and b == 3:
            nkv = nq // 2  # the first rows come before the first position
        q.append(nq)
        kv.append(nkv)
    return q, kv


def _seq_lens(case):
    rng = random.Random(case["shape"])
    return [_log_int(rng, case["len_lo"], case["len_hi"]) for _ in range(case["n_seq"])]


def _fork_plan(case):
    """(parent row, child row) pairs; rows from n_seq on are empty before."""
    rng = random.Random(case["shape"] + 1)
    return [rng.randrange(case["n_seq"]) for _ in range(case["n_child"])], [case["n_seq"] + i for i in range(case["n_child"])]


def _ended(case):
    rng = random.Random(case["shape"] + 2)
    n = case["n_seq"]
    return sorted(rng.sample(range(n), max(1, n // 2)))


def _cdiv(a, b):
    return -(-a // b)


def _visible(i, nq, nkv, window):
    """Positions [lo, hi) that new token i sees."""
    hi = max(0, nkv - nq + i + 1)
    lo = max(0, hi - window) if window > 0 else 0
    return lo, hi


def work(case):
    if case["op"] == "attend":
        q, kv = _lengths(case)
        pairs = reach = 0
        for nq, nkv in zip(q, kv):
            spans = [_visible(i, nq, nkv, case["window"]) for i in range(nq)]
            pairs += sum(hi - lo for lo, hi in spans)
            spans = [s for s in spans if s[1] > s[0]]
            reach += max(s[1] for s in spans) - min(s[0] for s in spans) if spans else 0
        rows = sum(q) * case["n_q"]
        return {"bytes": 4 * rows * case["hd"] + 4 * reach * case["n_kv"] * case["hd"] + (4 * rows if case["lse"] else 0),
                "flops": 4 * pairs * case["n_q"] * case["hd"]}
    if case["op"] == "rope_append":
        t = sum(_lengths(case)[0])
        heads = case["n_q"] + 2 * case["n_kv"]
        src = 4 if case["src"] == "f32" else 2
        return {"bytes": t * heads * case["hd"] * (src + 2), "flops": t * (case["n_q"] + case["n_kv"]) * (3 * case["n_rot"] + 4 * case["hd"])}
    page, lens = case["page"], _seq_lens(case)
    plane = case["planes"] * case["page_bytes"]
    held = [_cdiv(n, page) for n in lens]
    n_pages = _n_pages(case)
    if case["op"] == "fork":
        src, _ = _fork_plan(case)
        copies = sum(lens[s] % page != 0 for s in src)
        entries = sum(held[s] for s in src)
        return {"bytes": 2 * copies * plane + 4 * n_pages + 12 * entries, "flops": entries}
    live = sum(held) - sum(held[r] for r in _ended(case))
    order = _page_order(case)
    alive = torch.zeros(n_pages, dtype=torch.bool)
    at = 0
    ended = set(_ended(case))
    for r, h in enumerate(held):
        if r not in ended:
            alive[order[at:at + h]] = True
        at += h
    moves = int(alive[live:].sum())
    return {"bytes": 2 * moves * plane + 8 * n_pages + 8 * sum(held), "flops": sum(held)}


# --------------------------------------------------------------------------
# what a program has in hand


def _n_pages(case):
    lens = _seq_lens(case)
    return sum(_cdiv(n, case["page"]) for n in lens) + case["n_child"] + case["spare"]


def _page_order(case):
    """The order in which the pool's pages were given out."""
    return torch.randperm(_n_pages(case), generator=torch.Generator().manual_seed(case["shape"]))


def _rope_table(n_pos, n_rot, scaling, theta=1e6):
    """cos and sin of every position's angles, [n_pos, n_rot / 2, 2] fp32: plain,
    positions divided by 4 ("linear"), or slow pairs divided by 4 and fast
    ones kept, with a ramp between and both scaled by 0.1 ln 4 + 1 ("yarn")."""
    half = n_rot // 2
    j = torch.arange(half, dtype=torch.float64, device="cuda")
    freq = theta ** (-2.0 * j / n_rot)
    mul = 1.0
    if scaling == "linear":
        freq = freq / 4
    elif scaling == "yarn":
        turns = lambda r: n_rot * math.log(8192 / (2 * math.pi * r)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(0, math.floor(turns(32))), min(n_rot - 1, math.ceil(turns(1)))
        ramp = ((j - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        freq = freq / 4 * ramp + freq * (1 - ramp)
        mul = 0.1 * math.log(4) + 1
    a = torch.arange(n_pos, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.stack([a.cos() * mul, a.sin() * mul], -1).float().contiguous()


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + case["shape"])
    norm = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    st = {"case": case}
    if case["op"] in ("fork", "turnover"):
        page, lens, n_pages = case["page"], _seq_lens(case), _n_pages(case)
        rows, held = case["n_seq"] + case["n_child"], [_cdiv(n, case["page"]) for n in lens]
        table = torch.full((rows, max(held) + 1), -1, dtype=torch.int32)
        ref = torch.zeros(n_pages, dtype=torch.int32)
        order, at = _page_order(case).int(), 0
        for r, h in enumerate(held):
            table[r, :h] = order[at:at + h]
            ref[order[at:at + h].long()] = 1
            at += h
        st["table"], st["ref"], st["lens"] = table.cuda(), ref.cuda(), _ints(lens + [0] * case["n_child"])
        st["pool"] = torch.empty(case["planes"], n_pages, case["page_bytes"] // 2, dtype=torch.bfloat16, device="cuda")
        st["pool"].view(-1).normal_(generator=g)
        if case["op"] == "fork":
            src, dst = _fork_plan(case)
            st["src"], st["dst"] = _ints(src), _ints(dst)
        else:
            st["ended"] = _ints(_ended(case))
            st["work"] = [torch.empty_like(st[k]) for k in ("table", "ref", "lens")]
        if own:
            t = st["work"] if "work" in st else [st["table"], st["ref"], st["lens"]]
            st["pages"] = _m27b().PageSet(*t, page, pool=st["pool"])
        return st
    q_len, kv_len = _lengths(case)
    dt, page, n_kv, hd, n_q = _DTYPES[case["dtype"]], case["page"], case["n_kv"], case["hd"], case["n_q"]
    total = sum(q_len)
    cu = [0]
    for n in q_len:
        cu.append(cu[-1] + n)
    st["cu_q"], st["lens"] = _ints(cu), _ints(kv_len)
    cols = max(1, max(_cdiv(n, page) for n in kv_len))
    if case["op"] == "attend":
        # the sequences' pages lie anywhere in the pool, a few of it unused; a
        # slot past a sequence's last position holds whatever was there before
        need = sum(_cdiv(n, page) for n in kv_len)
        n_pages = need + 3
        order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(case["shape"] + int(seed))).int()
        table, at = torch.full((case["n_seq"], cols), -1, dtype=torch.int32), 0
        for b, n in enumerate(kv_len):
            h = _cdiv(n, page)
            table[b, :h] = order[at:at + h]
            at += h
        st["k"] = norm(n_pages, page, n_kv, hd).to(dt)
        st["v"] = norm(n_pages, page, n_kv, hd).to(dt)
        for b, n in enumerate(kv_len):
            if n % page:
                p = int(table[b, n // page])
                st["k"][p, n % page:] = float("nan")
                st["v"][p, n % page:] = float("inf")
        st["table"] = table.cuda()
        st["q"] = (1.5 * norm(total, n_q, hd)).to(dt)
        st["out"] = torch.zeros(total, n_q, hd, dtype=dt, device="cuda")
        st["lse"] = torch.zeros(total, n_q, device="cuda") if case["lse"] else None
        if own:
            m = _m27b()
            st["kv"] = m.PagedKV(st["k"], st["v"], st["table"])
            st["scratch"] = m.paged_attn_scratch(n_q, n_kv, hd)
        return st
    # rope_append: the pages that the new tokens touch are each sequence's own;
    # earlier ones are not looked at
    first = [(nkv - nq) // page for nq, nkv in zip(q_len, kv_len)]
    need = sum(_cdiv(n, page) - f for n, f in zip(kv_len, first))
    n_pages = need + 3
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(case["shape"] + int(seed))).int()
    table, at = torch.zeros(case["n_seq"], cols, dtype=torch.int32), 0
    for b, n in enumerate(kv_len):
        h = _cdiv(n, page) - first[b]
        table[b, first[b]:first[b] + h] = order[at:at + h]
        at += h
    st["table"] = table.cuda()
    st["k_pool"] = norm(n_pages, page, n_kv, hd).to(dt)
    st["v_pool"] = norm(n_pages, page, n_kv, hd).to(dt)
    src = _DTYPES[case["src"]]
    st["qkv"] = (3.0 * norm(total, n_q + 2 * n_kv, hd)).to(src)  # one projection's output
    st["q_norm"], st["k_norm"] = (1 + 0.2 * norm(hd), 1 + 0.2 * norm(hd)) if case["norm"] else (None, None)
    st["rope"] = _rope_table(max(kv_len), case["n_rot"], case["scaling"])
    st["q_out"] = torch.zeros(total, n_q, hd, dtype=dt, device="cuda")
    if own:
        st["kv"] = _m27b().PagedKV(st["k_pool"], st["v_pool"], st["table"])
    return st


# --------------------------------------------------------------------------
# one pass


def _token_rows(cu_q, lens, total):
    """(sequence, position) of each row of q."""
    t = torch.arange(total, device="cuda")
    b = torch.searchsorted(cu_q[1:].long(), t, right=True)
    return b, lens.long()[b] - cu_q.long()[b + 1] + t


def _attend_plain(st):
    case, q, table = st["case"], st["q"].float(), st["table"].long()
    lens, page, n_kv, n_q, hd = st["lens"].long(), case["page"], case["n_kv"], case["n_q"], case["hd"]
    n_seq, cols = table.shape
    total = q.shape[0]
    pos = torch.arange(cols * page, device="cuda")
    held = (pos < lens[:, None])[:, :, None, None]
    keys = torch.where(held, st["k"].float()[table.clamp(min=0)].view(n_seq, cols * page, n_kv, hd), 0.0)
    vals = torch.where(held, st["v"].float()[table.clamp(min=0)].view(n_seq, cols * page, n_kv, hd), 0.0)
    b, p = _token_rows(st["cu_q"], st["lens"], total)
    i = torch.arange(total, device="cuda") - st["cu_q"].long()[b]
    width = max(1, int((st["cu_q"][1:] - st["cu_q"][:-1]).max()))
    qp = torch.zeros(n_seq, width, n_q, hd, device="cuda")
    qp[b, i] = q
    at = torch.full((n_seq, width), -1, dtype=torch.long, device="cuda")
    at[b, i] = p
    qp = qp.view(n_seq, width, n_kv, n_q // n_kv, hd).permute(0, 2, 3, 1, 4).reshape(n_seq, n_kv, -1, hd)
    s = torch.matmul(qp, keys.permute(0, 2, 3, 1)).mul_(1 / math.sqrt(hd)).view(n_seq, n_kv, n_q // n_kv, width, -1)
    see = pos <= at[:, :, None]
    if case["window"]:
        see &= pos > at[:, :, None] - case["window"]
    s.masked_fill_(~see[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = s.sub_(top.clamp(min=-1e30)).exp_()
    total_e = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(n_seq, n_kv, -1, cols * page), vals.transpose(1, 2)).view(n_seq, n_kv, -1, width, hd)
    o = o / torch.where(total_e > 0, total_e, 1.0)
    out = o.permute(0, 3, 1, 2, 4).reshape(n_seq, width, n_q, hd)[b, i].to(st["q"].dtype)
    if not case["lse"]:
        return [out]
    lse = (top + total_e.log())[..., 0].permute(0, 3, 1, 2).reshape(n_seq, width, n_q)[b, i]
    return [out, lse]


def _rope_plain(st):
    case, n_q, n_kv, page = st["case"], st["case"]["n_q"], st["case"]["n_kv"], st["case"]["page"]
    x = st["qkv"].float()
    b, p = _token_rows(st["cu_q"], st["lens"], x.shape[0])
    cos, sin = st["rope"][p][:, None, :, 0], st["rope"][p][:, None, :, 1]

    def turn(x, w):
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        r, rest = x[..., :case["n_rot"]], x[..., case["n_rot"]:]
        if case["interleaved"]:
            u, v = r[..., 0::2], r[..., 1::2]
            r = torch.stack([u * cos - v * sin, u * sin + v * cos], -1).flatten(-2)
        else:
            u, v = r.chunk(2, -1)
            r = torch.cat([u * cos - v * sin, u * sin + v * cos], -1)
        return torch.cat([r, rest], -1)

    q, k, v = x[:, :n_q], x[:, n_q:n_q + n_kv], x[:, n_q + n_kv:]
    at = st["table"].long()[b, p // page], p % page
    st["k_pool"][at] = turn(k, st["k_norm"]).to(st["k_pool"].dtype)
    st["v_pool"][at] = v.to(st["v_pool"].dtype)
    return [turn(q, st["q_norm"]).to(st["q_out"].dtype), st["k_pool"], st["v_pool"]]


def _drop_plain(table, ref, lens, rows, page):
    cols = torch.arange(table.shape[1], device="cuda")
    held = cols < ((lens[rows] + page - 1) // page)[:, None]
    ids = table[rows][held].long()
    ref.index_add_(0, ids, torch.full_like(ids, -1, dtype=torch.int32))
    table[rows] = table[rows].masked_fill(held, -1)
    lens[rows] = 0


def _fork_plain(st):
    page, table, ref, lens = st["case"]["page"], st["table"], st["ref"], st["lens"]
    src, dst = st["src"].long(), st["dst"].long()
    n = lens[src]
    cols = torch.arange(table.shape[1], device="cuda")
    new = table[src].masked_fill(cols >= ((n + page - 1) // page)[:, None], -1)
    part = (n % page != 0).nonzero()[:, 0]
    fresh = (ref == 0).nonzero()[:part.shape[0], 0]
    last = (n[part] // page).long()
    old = new[part, last].long()
    new[part, last] = fresh.int()
    st["pool"][:, fresh] = st["pool"][:, old]
    ids = new[new >= 0].long()
    ref.index_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))
    table[dst], lens[dst] = new, n
    grown = [table.clone(), ref.clone(), lens.clone()]
    _drop_plain(table, ref, lens, dst, page)
    return grown + [table, ref, lens, st["pool"]]


def _turnover_plain(st):
    page = st["case"]["page"]
    table, ref, lens = st["work"]
    _drop_plain(table, ref, lens, st["ended"].long(), page)
    live = (ref > 0).nonzero()[:, 0]
    src = live[live >= live.shape[0]]
    dst = (ref[:live.shape[0]] == 0).nonzero()[:, 0]
    st["pool"][:, dst] = st["pool"][:, src]
    ref[dst] = ref[src]
    ref[src] = 0
    new = torch.arange(ref.shape[0], device="cuda", dtype=torch.int32)
    new[src] = dst.int()
    table.copy_(torch.where(table >= 0, new[table.clamp(min=0).long()], table))
    return [table, ref, lens, st["pool"]]


def run(st):
    case = st["case"]
    if case["op"] == "turnover":
        # the same pages are freed and moved in every pass
        for to, name in zip(st["work"], ("table", "ref", "lens")):
            to.copy_(st[name])
    if not own:
        return {"attend": _attend_plain, "rope_append": _rope_plain, "fork": _fork_plain,
                "turnover": _turnover_plain}[case["op"]](st)
    m = _m27b()
    if case["op"] == "attend":
        m.paged_attn(st["kv"], st["q"], st["cu_q"], st["lens"], st["out"], window=case["window"], lse=st["lse"],
                     scratch=st["scratch"])
        return [st["out"], st["lse"]] if case["lse"] else [st["out"]]
    if case["op"] == "rope_append":
        n_q, n_kv, x = case["n_q"], case["n_kv"], st["qkv"]
        m.rope_append(st["kv"], x[:, :n_q], x[:, n_q:n_q + n_kv], x[:, n_q + n_kv:], st["cu_q"], st["lens"], st["rope"],
                      st["q_out"], interleaved=case["interleaved"], q_norm=st["q_norm"], k_norm=st["k_norm"], eps=1e-6)
        return [st["q_out"], st["k_pool"], st["v_pool"]]
    pages = st["pages"]
    if case["op"] == "fork":
        pages.fork(st["src"], st["dst"])
        grown = [st["table"].clone(), st["ref"].clone(), st["lens"].clone()]
        pages.free(st["dst"])
        return grown + [st["table"], st["ref"], st["lens"], st["pool"]]
    pages.free(st["ended"])
    pages.compact()
    return st["work"] + [st["pool"]]


# --------------------------------------------------------------------------
# the definitions in 64 bits


def _attend_exact(case, st):
    q_len, kv_len = _lengths(case)
    n_q, n_kv, hd, page, group = case["n_q"], case["n_kv"], case["hd"], case["page"], case["n_q"] // case["n_kv"]
    out = torch.zeros(sum(q_len), n_q, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((sum(q_len), n_q), -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for b, (nq, nkv) in enumerate(zip(q_len, kv_len)):
        ids = st["table"][b, :_cdiv(nkv, page)].long()
        key = st["k"][ids].reshape(-1, n_kv, hd)[:nkv].double()
        val = st["v"][ids].reshape(-1, n_kv, hd)[:nkv].double()
        for lo in range(0, nq if nkv else 0, 512):
            rows = range(lo, min(nq, lo + 512))
            spans = torch.tensor([_visible(i, nq, nkv, case["window"]) for i in rows], device="cuda")
            pos = torch.arange(nkv, device="cuda")
            hide = (pos < spans[:, :1]) | (pos >= spans[:, 1:])
            for j in range(n_kv):
                x = st["q"][at + lo:at + lo + len(rows), j * group:(j + 1) * group].double()
                s = torch.einsum("thd,pd->thp", x, key[:, j]) / math.sqrt(hd)
                s = s.masked_fill(hide[:, None], -math.inf)
                z = torch.logsumexp(s, -1)
                w = torch.exp(s - z.masked_fill(z == -math.inf, 0.0)[..., None])
                out[at + lo:at + lo + len(rows), j * group:(j + 1) * group] = torch.einsum("thp,pd->thd", w, val[:, j])
                lse[at + lo:at + lo + len(rows), j * group:(j + 1) * group] = z
        at += nq
    return [out, lse] if case["lse"] else [out]


def _rope_exact(case, st):
    q_len, kv_len = _lengths(case)
    n_q, n_kv, half = case["n_q"], case["n_kv"], case["n_rot"] // 2
    x = st["qkv"].double()
    k_pool, v_pool = st["k_pool"].double(), st["v_pool"].double()
    seq = [(b, kv_len[b] - q_len[b] + i) for b in range(case["n_seq"]) for i in range(q_len[b])]
    row = torch.tensor([s[0] for s in seq], device="cuda")
    pos = torch.tensor([s[1] for s in seq], device="cuda")
    factor = torch.view_as_complex(st["rope"].double()[pos].contiguous())[:, None]
    d = torch.arange(half, device="cuda")
    first, second = (2 * d, 2 * d + 1) if case["interleaved"] else (d, d + half)

    def turned(y, w):
        if w is not None:
            y = y * torch.rsqrt(y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + 1e-6) * w.double()
        z = torch.complex(y[..., first], y[..., second]) * factor
        y = y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    page = st["table"].long()[row, pos // case["page"]]
    k_pool[page, pos % case["page"]] = turned(x[:, n_q:n_q + n_kv], st["k_norm"])
    v_pool[page, pos % case["page"]] = x[:, n_q + n_kv:]
    return [turned(x[:, :n_q], st["q_norm"]), k_pool, v_pool]


def _pages_exact(case, st):
    """Page by page, with lists; the pool's values are copies."""
    page, pool = case["page"], st["pool"]
    table, ref, lens = st["table"].tolist(), st["ref"].tolist(), st["lens"].tolist()

    def drop(rows):
        for r in rows:
            for i in range(_cdiv(lens[r], page)):
                ref[table[r][i]] -= 1
                table[r][i] = -1
            lens[r] = 0

    def move(pairs):
        if pairs:
            a, b = (torch.tensor(v, device="cuda") for v in zip(*pairs))
            pool[:, b] = pool[:, a]

    if case["op"] == "fork":
        src, dst = _fork_plan(case)
        free = iter([p for p, n in enumerate(ref) if n == 0])
        pairs = []
        for s, d in zip(src, dst):
            lens[d] = lens[s]
            for i in range(_cdiv(lens[s], page)):
                p = table[s][i]
                if (i + 1) * page > lens[s]:
                    p = next(free)
                    pairs.append((table[s][i], p))
                table[d][i] = p
                ref[p] += 1
        move(pairs)
        grown = [_ints(table), _ints(ref), _ints(lens)]
        drop(dst)
        return grown + [_ints(table), _ints(ref), _ints(lens), pool]
    drop(_ended(case))
    live = sum(n > 0 for n in ref)
    to = {}
    holes = iter([p for p in range(live) if ref[p] == 0])
    for p in range(live, len(ref)):
        if ref[p] > 0:
            to[p] = next(holes)
            ref[to[p]], ref[p] = ref[p], 0
    move(list(to.items()))
    table = [[to.get(p, p) for p in r] for r in table]
    return [_ints(table), _ints(ref), _ints(lens), pool]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attend":
        return _attend_exact(case, st)
    if case["op"] == "rope_append":
        return _rope_exact(case, st)
    return _pages_exact(case, st)
