"""Serving on the paged 4-bit KV cache: two prompts, samples forked from them, drafts verified and trimmed, rows
retired and the pool compacted.  Queries, keys and values are random; every attention is compared with a dense one
over the rows as the cache holds them.

    python win-directml-java_b200/examples/paged_kv4.py
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import b200attn  # noqa: E402

LAYERS, HQ, HKV, D, PAGE, THETA = 2, 8, 2, 64, 32, 1e6
SCALE = 1 / math.sqrt(D)


class Server:
    """The rows of a batch: one page table and one count per page for all layers, their lengths, and (for the
    comparison alone) each row's keys and values as the cache holds them."""

    def __init__(self, rows, num_pages, max_pages, dtype=torch.bfloat16, seed=0):
        self.ctx = b200attn.Context(0)
        self.rows, self.dtype = rows, dtype
        self.gen = torch.Generator("cuda").manual_seed(seed)
        slab = b200attn.kv4_page_bytes(HKV, D, PAGE) // HKV
        self.pages = torch.zeros(LAYERS, num_pages, HKV, slab, dtype=torch.uint8, device="cuda")
        self.table = torch.full((rows, max_pages), -1, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(num_pages, dtype=torch.int32, device="cuda")
        self.counts = torch.zeros(2, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.held = [[torch.zeros(2, 0, HKV, D, device="cuda") for _ in range(rows)] for _ in range(LAYERS)]
        self.worst = 0.0  # largest difference from dense attention
        self.worst_of_bound = 0.0  # the same, as a share of what roundings allow that element

    def step(self, new):
        """Appends and attends new[row] tokens per row (a chunk, a draft, one token, or none)."""
        new_lens = torch.tensor(new, dtype=torch.int32, device="cuda")
        b200attn.pages_reserve(self.ctx, self.table, self.refs, self.lens, new_lens, self.pages, PAGE, self.counts)
        if int(self.counts[1]):
            raise RuntimeError(f"{int(self.counts[1])} pages are missing")
        T = max(new)
        for layer in range(LAYERS):
            fused = torch.randn(self.rows, T, (HQ + 2 * HKV) * D, generator=self.gen, device="cuda").to(self.dtype)
            heads = fused.view(self.rows, T, HQ + 2 * HKV, D)  # a projection's [Q|K|V] rows
            q, k, v = heads[:, :, :HQ], heads[:, :, HQ:HQ + HKV], heads[:, :, HQ + HKV:]
            out = torch.empty(self.rows, T, HQ, D, dtype=self.dtype, device="cuda")
            kh, vh = (torch.empty(self.rows, T, HKV, D, dtype=self.dtype, device="cuda") for _ in range(2))
            b200attn.kv4_decode(self.ctx, q, k, v, self.pages[layer], self.table, self.lens, out, SCALE,
                                new_lens=new_lens, rope_theta=THETA, k_held=kh, v_held=vh)
            for row, n in enumerate(new):
                fresh = torch.stack([kh[row, :n], vh[row, :n]]).float()
                self.held[layer][row] = torch.cat([self.held[layer][row], fresh], 1)
                if n:
                    self.compare(layer, row, q[row, :n], out[row, :n])
        self.ctx.check_device_status()
        self.lens += new_lens

    def keep(self, lens):
        """Trims rows to the positions that were accepted (0: the row leaves)."""
        self.lens.copy_(torch.tensor(lens, dtype=torch.int32, device="cuda"))
        b200attn.pages_free(self.ctx, self.table, self.refs, None, self.lens, PAGE)
        for layer in self.held:
            for row, n in enumerate(lens):
                layer[row] = layer[row][:, :n]

    def fork(self, parents):
        """Row i goes on as a copy of row parents[i] (-1: empty); pages are shared until one writes to them."""
        b200attn.pages_fork(self.ctx, self.table, self.refs, torch.tensor(parents, dtype=torch.int32, device="cuda"))
        self.lens = torch.stack([self.lens[p] if p >= 0 else self.lens.new_zeros(()) for p in parents])
        self.held = [[layer[p] if p >= 0 else layer[0][:, :0] for p in parents] for layer in self.held]

    def compact(self):
        b200attn.pages_compact(self.ctx, self.table, self.refs, self.pages, self.counts)
        return self.counts.tolist()

    def compare(self, layer, row, q, out):
        k, v = self.held[layer][row].double()
        n, total = q.shape[0], k.shape[0]
        pos = torch.arange(total - n, total, device="cuda")
        angle = pos[:, None].double() / THETA ** (torch.arange(0, D, 2, device="cuda").double() / D)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        a, b = q.double().split(D // 2, -1)
        q = torch.cat([a * c - b * s, b * c + a * s], -1).view(n, HKV, HQ // HKV, D)
        score = SCALE * torch.einsum("nhgd,khd->nhgk", q, k)
        score.masked_fill_((torch.arange(total, device="cuda") > pos[:, None])[:, None, None], -math.inf)
        p = score.softmax(-1)
        want = torch.einsum("nhgk,khd->nhgd", p, v)
        # bf16 rounds the held keys and values and the output by 2^-9 each, the kernels round q, P, P s and a
        # chunk's rows by 2^-11 each: `off` of a score, which moves its weight by as much, and of a value
        off = (2 ** -9 + 2 * 2 ** -11) * SCALE * torch.einsum("nhgd,khd->nhgk", q.abs(), k.abs())
        bound = 2 ** -8 * want.abs() + (2 ** -9 + 4 * 2 ** -11 + 1e-5) * torch.einsum("nhgk,khd->nhgd", p, v.abs())
        for h in range(HKV):  # sum_j p_j off_j |v_j - o|
            far = (v[None, None, :, h] - want[:, h, :, None]).abs()
            bound[:, h] += torch.einsum("ngk,ngkd->ngd", p[:, h] * off[:, h], far)
        err = (out.double().view_as(want) - want).abs()
        self.worst = max(self.worst, float(err.max()))
        self.worst_of_bound = max(self.worst_of_bound, float((err / bound).max()))


def main():
    s = Server(rows=6, num_pages=48, max_pages=8)
    s.step([150, 45, 0, 0, 0, 0])                      # two prompts
    s.fork([0, 0, 0, 1, 1, -1])                        # three samples of the first, two of the second
    s.step([1, 1, 1, 1, 1, 0])                         # each writes: the shared last pages are copied
    for accepted in ([4, 1, 2, 5, 3, 0], [1, 5, 1, 2, 2, 0]):
        before = s.lens.tolist()
        s.step([5, 5, 5, 5, 5, 0])                     # drafts of five tokens are verified at once
        s.keep([n + a for n, a in zip(before, accepted)])
    lens = s.lens.tolist()
    s.keep([lens[0], 0, lens[2], 0, lens[4], 0])       # two samples are done
    used, moved = s.compact()
    s.fork([0, 2, 4, -1, -1, -1])                      # the others move to the front
    s.step([1, 1, 1, 70, 0, 0])                        # they go on beside a new prompt
    s.step([1, 1, 1, 1, 0, 0])
    print(f"rows of {s.lens.tolist()} tokens on {int((s.refs > 0).sum())} pages ({used} after compaction, which moved "
          f"{moved}); largest difference from dense attention {s.worst:.2e}, {s.worst_of_bound:.0%} of its bound")
    return s


if __name__ == "__main__":
    main()
