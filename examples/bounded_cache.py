"""A batch served from a bounded 8-bit cache.

    python examples/bounded_cache.py [--steps N] [--budget N]

Prompts are packed row after row and attended at once (`PackedPlan`), their
keys and values go to FP8 pages (`F8Plan.write`), and decode steps attend to
the pages and count the weight that each slot receives.  A sequence that
outgrows its budget keeps its newest slots and those with the largest
counters, per head, in new pages (`F8Plan.evict`), and its old pages are
freed.  Random projections stand in for a model's.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import molot_b200 as mb  # noqa: E402


class Batch:
    """Sequences of one layer in a pager's pages, and the step that grows them."""

    def __init__(self, nq=32, nkv=8, d=128, page_size=16, pages=4096, max_seqs=16, softcap=50.0):
        self.nq, self.nkv, self.d, self.softcap = nq, nkv, d, softcap
        self.scale = d ** -0.5
        self.pager = mb.Pager(1, nkv, d, page_size, pages, max_seqs, pages, dtype="f8b")
        self.plan, self.packed = mb.F8Plan(), mb.PackedPlan()
        self.seqs = []

    def _layer(self, seqs):
        table, lens = self.pager.tables(seqs)
        return self.pager.f8_layer(0, torch.from_numpy(table).cuda()), lens

    def split(self, qkv):
        """The query, key and value parts of a projection [rows][nq + 2 nkv][d]."""
        return (qkv[:, :self.nq], qkv[:, self.nq:self.nq + self.nkv], qkv[:, self.nq + self.nkv:])

    def prefill(self, qkv, lens):
        """Attention of whole prompts; their rows enter the cache."""
        q, k, v = self.split(qkv)
        out = torch.empty(q.shape, device="cuda", dtype=q.dtype)
        self.packed.build(self.nq, self.nkv, self.d, lens)
        self.packed.attend(q, k, v, out, self.scale, softcap=self.softcap)
        new = [self.pager.add(n) for n in lens]
        self.seqs += new
        layer, n = self._layer(new)
        self.plan.build(self.nq, self.nkv, self.d, n, new_lens=n)
        self.plan.write(layer, k, v)
        return out

    def step(self, qkv):
        """One token per sequence: append, attend, count."""
        q, k, v = self.split(qkv)
        out = torch.empty(q.shape, device="cuda", dtype=q.dtype)
        for s in self.seqs:
            self.pager.grow(s)
        layer, lens = self._layer(self.seqs)
        self.plan.build(self.nq, self.nkv, self.d, lens)
        self.plan.write(layer, k, v)
        self.plan.decode(layer, q, out, self.scale, softcap=self.softcap,
                         weight_out=layer.tensors[4])
        return out

    def bound(self, budget, recent):
        """Brings sequences that outgrew the budget back to it."""
        long = [i for i, s in enumerate(self.seqs) if self.pager.length(s) > budget]
        if not long:
            return []
        old = [self.seqs[i] for i in long]
        src, lens = self._layer(old)
        new = [self.pager.add(budget) for _ in old]
        dst, _ = self._layer(new)
        kept = torch.empty(len(old), self.nkv, budget, dtype=torch.int32, device="cuda")
        self.plan.build(self.nq, self.nkv, self.d, lens)
        self.plan.evict(src, dst, budget, recent, kept)
        for i, s, t in zip(long, old, new):
            self.pager.free(s)  # its pages are written again only by later work on this stream
            self.seqs[i] = t
        return long

    def close(self):
        self.plan.check()
        self.packed.check()
        for x in (self.plan, self.packed, self.pager):
            x.close()


def main(steps=64, budget=1024, recent=128, prompts=(900, 1000, 1500, 37), every=16):
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    batch = Batch()
    rows = batch.nq + 2 * batch.nkv

    def project(n):
        return torch.randn(n, rows, batch.d, device="cuda", generator=g).bfloat16()

    out = batch.prefill(project(sum(prompts)), list(prompts))
    print(f"prefilled {len(prompts)} prompts, {sum(prompts)} rows, |o| {out.float().norm():.2f}")
    for i in range(steps):
        out = batch.step(project(len(batch.seqs)))
        if (i + 1) % every == 0:
            moved = batch.bound(budget, recent)
            lens = [batch.pager.length(s) for s in batch.seqs]
            print(f"step {i + 1}: slots {lens}, evicted from {len(moved)}, "
                  f"free pages {batch.pager.free_pages()}, |o| {out.float().norm():.2f}")
    lens = [batch.pager.length(s) for s in batch.seqs]
    batch.close()
    return lens, out


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--budget", type=int, default=1024)
    a = ap.parse_args()
    main(steps=a.steps, budget=a.budget)
