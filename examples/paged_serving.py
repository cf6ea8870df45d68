"""Several sequences over one paged key/value cache: prompts in chunks, one
prompt answered several ways, answers dropped, pages moved together.

    python examples/paged_serving.py

A small attention stack (random weights, no vocabulary): every layer projects
the hidden states, m27b.rope_append normalises and rotates q and k and puts k
and v into the cache, m27b.paged_attn attends over it.  One function, step(),
takes any mix of prompt chunks and single tokens; PageSet gives the sequences
their pages.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mono-qwen27_b200"))
import m27b  # noqa: E402


class Stack:
    """n_layers attention layers over a cache of n_pages pages."""

    def __init__(self, n_layers=4, hidden=1024, n_q=16, n_kv=8, head_dim=128, n_pages=400, page_size=16, max_seqs=12,
                 max_len=2048, dtype=torch.bfloat16, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        w = lambda *s: torch.randn(*s, generator=g, device="cuda") / s[-1] ** 0.5  # noqa: E731
        self.n_q, self.n_kv, self.hd, self.hidden = n_q, n_kv, head_dim, hidden
        self.w_qkv = [w((n_q + 2 * n_kv) * head_dim, hidden) for _ in range(n_layers)]
        self.w_out = [w(hidden, n_q * head_dim) for _ in range(n_layers)]
        self.norm = torch.ones(head_dim, device="cuda")
        self.rope = m27b.rope_table(max_len, head_dim // 2, 1e6, kind=m27b.ROPE_YARN, factor=2.0, original_ctx=max_len // 2)
        # planes 2 l and 2 l + 1: layer l's keys and values
        pool = torch.zeros(2 * n_layers, n_pages, page_size, n_kv, head_dim, dtype=dtype, device="cuda")
        self.pages = m27b.PageSet.empty(max_seqs, max_len // page_size, n_pages, page_size, pool)
        self.kv = [m27b.PagedKV(pool[2 * i], pool[2 * i + 1], self.pages.table) for i in range(n_layers)]
        self.scratch = m27b.paged_attn_scratch(n_q, n_kv, head_dim)
        self.dtype = dtype

    def step(self, rows, lens, x):
        """The next tokens of the sequences in `rows`: lens, how many each; x,
        their hidden states one after the other.  Returns the new ones."""
        rows_t, lens_t = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (rows, lens))
        cu = torch.zeros(len(rows) + 1, dtype=torch.int32, device="cuda")
        cu[1:] = lens_t.cumsum(0)
        self.pages.resize(rows_t, self.pages.lens[rows_t.long()] + lens_t)
        self.pages.check()  # refused: lens are the old ones, and the append would overwrite the last positions
        q = torch.empty(len(x), self.n_q, self.hd, dtype=self.dtype, device="cuda")
        o = torch.empty_like(q)
        for kv, w_qkv, w_out in zip(self.kv, self.w_qkv, self.w_out):
            qkv = (torch.nn.functional.rms_norm(x, (self.hidden,)) @ w_qkv.t()).view(len(x), -1, self.hd)
            n = self.n_q + self.n_kv
            m27b.rope_append(kv, qkv[:, :self.n_q], qkv[:, self.n_q:n], qkv[:, n:], cu, self.pages.lens, self.rope, q,
                             q_norm=self.norm, k_norm=self.norm, rows=rows_t)
            m27b.paged_attn(kv, q, cu, self.pages.lens, o, self.scratch, rows=rows_t)
            x = x + o.view(len(x), -1).float() @ w_out.t()
        return x

    def fork(self, parent, children):
        i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        self.pages.fork(i([parent] * len(children)), i(children))
        self.pages.check()

    def free(self, rows):
        self.pages.free(torch.tensor(rows, dtype=torch.int32, device="cuda"))


def main():
    torch.manual_seed(1)
    s = Stack()
    tokens = lambda n: torch.randn(n, s.hidden, device="cuda")  # noqa: E731
    # three prompts, the longest in two chunks, the second beside the others
    a, b, c = tokens(700), tokens(333), tokens(40)
    s.step([0], [400], a[:400])
    y = s.step([0, 1, 2], [300, 333, 40], torch.cat([a[400:], b, c]))
    # prompt 1 answered three ways: the same first token, then another each
    s.fork(1, [3, 4, 5])
    one = y[632:633]
    y = s.step([1, 3, 4, 5], [1] * 4, one.repeat(4, 1))
    same = bool((y == y[0]).all())
    y = s.step([1, 3, 4, 5], [1] * 4, tokens(4))
    # the same answer without a fork: its prompt again, in another row
    s.step([6], [333], b)
    z = s.step([6], [1], one)
    for _ in range(20):
        y = s.step([1, 3, 4, 5], [1] * 4, y)
    used = int((s.pages.ref > 0).sum())
    s.free([0, 3, 4])
    live = torch.zeros(1, dtype=torch.int32, device="cuda")
    s.pages.compact(n_live=live)
    y = s.step([1, 5], [1, 1], y[[0, 3]])  # what is left goes on
    s.pages.check()
    assert m27b.device_status() == 0 and same and bool(torch.isfinite(y).all())
    print(f"pages in use {used}, {int(live)} after two answers and a prompt ended; highest page {int(s.pages.table.max())}")
    return one, z, y


if __name__ == "__main__":
    main()
