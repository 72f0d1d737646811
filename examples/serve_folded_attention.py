"""A folded stack's attention block, served: prompts, then decoding, over a
4-bit paged cache.

The q / k / v / o projections are this library's folded FP4 sparse layers
(sili__new_b200.folded); page tables, rotary positions, the cache and the
attention over it are sili__new_b200.serving.  Requests of different lengths
share one cache; one is finished on the way and its pages are reused.

    python examples/serve_folded_attention.py [--hidden 512 --heads 8 ...]

With --check each step's attention is compared with a plain one in 64 bits
over the values that the cache holds.
"""
from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from sili__new_b200 import SparseLinearLayer, folded, serving  # noqa: E402


class ServedAttention:
    """One attention block of a folded stack and the requests it serves."""

    def __init__(self, hidden, heads, kv_heads, dim, folds, density, requests, pages, page, most_positions, scaling=None,
                 seed=0):
        self.hidden, self.heads, self.kv_heads, self.dim = hidden, heads, kv_heads, dim
        shapes = {"q_proj": (hidden, heads * dim), "k_proj": (hidden, kv_heads * dim),
                  "v_proj": (hidden, kv_heads * dim), "o_proj": (heads * dim, hidden)}
        self.stack = folded.FoldedStack(shapes, folds, 0, 1, lambda i, o, n: SparseLinearLayer(i, o, n, 1, 0))
        for k, (name, (n_in, n_out)) in enumerate(shapes.items()):
            ptrs, idx, vals, nnz = folded.synthetic_shard(n_in, n_out, folds, density, 0, n_out, seed + k, "cuda")
            self.stack.load(name, ptrs, idx, vals, nnz, folded.SYNTHETIC_VALUE_SCALE)
        self.cache = serving.KVCache4(pages, page, kv_heads, dim)
        self.ring, self.pool = serving.page_pool(pages)
        self.table = torch.full((requests, pages), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.cos, self.sin = serving.rotary_table(most_positions, dim, scaling=scaling)

    def step(self, x, fresh, most_new):
        """x [tokens, hidden]: the new tokens of all requests back to back,
        fresh[r] of them request r's; rows past the last are padding.
        Returns the block's output [tokens, hidden]."""
        tokens = x.shape[0]
        stream = torch.cuda.current_stream()
        out = self.stack.forward_group(["q_proj", "k_proj", "v_proj"], {n: x for n in ("q_proj", "k_proj", "v_proj")}, stream)
        q = out["q_proj"].view(tokens, self.heads, self.dim)
        k = out["k_proj"].view(tokens, self.kv_heads, self.dim)
        v = out["v_proj"].view(tokens, self.kv_heads, self.dim)
        t = serving.page_tables(self.lens, fresh, self.table, self.ring, self.pool, self.cache.page, tokens)
        self.lens, self.pool = t.lens, t.pool
        q = serving.cache_append(k, v, self.cache.codes, self.cache.scales, t.slots, cos=self.cos, sin=self.sin,
                                 positions=t.positions, q=q)
        y = serving.cache_attention(q, self.cache.codes, self.cache.scales, self.table, t.lens, starts=t.starts,
                                    most_new=most_new)
        self.last = (q, t, y)
        return self.stack.forward_device("o_proj", y.view(tokens, -1), stream)

    def finish(self, done):
        """The requests of the bool mask are over: their pages are free again."""
        self.pool = serving.release_pages(done, self.lens, self.table, self.ring, self.pool, self.cache.page)

    def error(self):
        """Largest deviation of the last step's attention from a plain one in
        64 bits over the cached values, over the largest output."""
        q, t, y = self.last
        starts, worst = t.starts.tolist(), 0.0
        page = self.cache.page
        for r, length in enumerate(t.lens.tolist()):
            n = starts[r + 1] - starts[r]
            if not n:
                continue
            at = torch.arange(length, device="cuda")
            slots = self.table[r].long()[at // page] * page + at % page
            k, v = (a.double() for a in serving.cache_read(self.cache.codes, self.cache.scales, slots))
            rows = q[starts[r]:starts[r + 1]].double().view(n, self.kv_heads, -1, self.dim)
            s = torch.einsum("nhgd,lhd->hgnl", rows, k) / math.sqrt(self.dim)
            s = s.masked_fill(at[None, :] > torch.arange(length - n, length, device="cuda")[:, None], float("-inf"))
            want = torch.einsum("hgnl,lhd->nhgd", s.softmax(-1), v).reshape(n, self.heads, self.dim)
            got = y[starts[r]:starts[r + 1]].double()
            worst = max(worst, float((got - want).abs().max() / want.abs().max()))
        return worst


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("hidden", 512), ("heads", 8), ("kv-heads", 2), ("dim", 64), ("folds", 2), ("page", 16),
                        ("pages", 64), ("decode", 20)):
        ap.add_argument("--" + name, type=int, default=value)
    ap.add_argument("--density", type=float, default=0.1)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args(argv)
    prompts = [37, 5, 120, 64]
    block = ServedAttention(a.hidden, a.heads, a.kv_heads, a.dim, a.folds, a.density, len(prompts), a.pages, a.page, 4096,
                            scaling={"type": "wavelength", "factor": 4.0, "original": 1024})
    gen = torch.Generator(device="cuda").manual_seed(1)
    worst = 0.0

    def run(fresh, most_new):
        nonlocal worst
        fresh = torch.tensor(fresh, dtype=torch.int32, device="cuda")
        tokens = -(-int(fresh.sum()) // 8) * 8           # padded to a multiple of 8
        y = block.step(torch.randn(tokens, a.hidden, generator=gen, device="cuda"), fresh, most_new)
        if a.check:
            worst = max(worst, block.error())
        return y

    run(prompts, max(prompts))
    for i in range(a.decode):
        if i == a.decode // 2:
            block.finish(torch.tensor([False, True, True, False], device="cuda"))
            run([1, 30, 0, 1], 30)                       # a new prompt in a freed row, beside decoding
        y = run([1, 1, 0, 1], 1)
    serving.check_attention()
    print(f"served {len(prompts)} prompts and {a.decode} decode steps: lengths {block.lens.tolist()}, "
          f"{int(block.pool[0] - block.pool[1]) + a.pages} of {a.pages} pages in use, output {list(y.shape)}"
          + (f", attention within {worst:.1e} of 64 bits" if a.check else ""))
    return block, worst


if __name__ == "__main__":
    main()
