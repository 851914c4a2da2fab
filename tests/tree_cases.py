"""Inputs and plain forms for the tests of tree_layout, paged_tree, sample_tokens, accept_tree and copy_blocks."""

from __future__ import annotations

import math
import random

import torch

from tests.chunk_cases import LAYER, Chunk, half_step


# ------------------------------------------------------------------------------------------------ trees
def grown(nodes: int, seed: int, roots: int = 1, line: bool = False) -> list[int]:
    """Parents of a random tree; its first ``roots`` nodes have none. ``line``: each node follows the one before."""
    rng = random.Random(seed)
    return [-1 if i < roots else i - 1 if line else rng.randrange(i) for i in range(nodes)]


def lines_of(parents: list[int]) -> list[list[int]]:
    """Each node and its ancestors."""
    lines = []
    for i, p in enumerate(parents):
        lines.append(([] if p < 0 else lines[p]) + [i])
    return lines


def packed(lines: list[list[int]], words: int) -> torch.Tensor:
    """int64 [nodes, words] with each line's bits."""
    rows = []
    for line in lines:
        bits = [0] * words
        for j in line:
            bits[j // 64] |= 1 << j % 64
        rows.append([b - (1 << 64) if b >> 63 else b for b in bits])
    return torch.tensor(rows, dtype=torch.int64).reshape(-1, words)


def unpacked(masks: torch.Tensor) -> torch.Tensor:
    """bool [nodes, 64 words]."""
    return (masks[..., None] >> torch.arange(64) & 1).bool().flatten(-2)


# --------------------------------------------------------------------------------------------- attention
class Tree(Chunk):
    """A call of paged_tree: sequences of ``(start, parents)``."""

    def __init__(self, seqs, heads, kv_heads, dim, dtype, block_size, words=None, **more):
        super().__init__([(s, len(p)) for s, p in seqs], heads, kv_heads, dim, dtype, block_size, **more)
        self.parents = [p for _, p in seqs]
        words = words or -(-max([1] + [len(p) for p in self.parents]) // 64)
        # Rows of no sequence: any bits.
        self.masks = torch.full((self.q.size(0), words), -1, dtype=torch.int64)
        for b, p in enumerate(self.parents):
            if p:
                self.masks[int(self.cu[b]) : int(self.cu[b + 1])] = packed(lines_of(p), words)

    def seen(self, b):
        """bool [new, start + new]."""
        s, n = self.seqs[b]
        bits = unpacked(self.masks[int(self.cu[b]) : int(self.cu[b + 1])])
        bits = torch.nn.functional.pad(bits, (0, max(0, n - bits.size(1))))[:, :n].tril()
        return torch.cat([torch.ones(n, s, dtype=torch.bool), bits], 1)

    def expected(self, scale=None):
        """``Chunk.expected`` with the rows' masks in place of the causal one; rows that see nothing are zero, exactly."""
        scale = 1 / math.sqrt(self.dim) if scale is None else scale
        out = torch.full(self.q.shape, math.nan, dtype=torch.float64)
        bound = out.clone()
        group, step = self.heads // self.kv_heads, half_step(self.dtype)
        for b, (s, n) in enumerate(self.seqs):
            if n == 0:
                continue
            k, v = self.keys_values(b)
            r0 = int(self.cu[b])
            seen = self.seen(b)
            some = seen.any(-1, keepdim=True)
            for h in range(self.heads):
                q, kh = self.q[r0 : r0 + n, h].double(), k[:, h // group]
                vh = v[:, h // group]
                x = torch.where(seen, q @ kh.t() * scale, -math.inf)
                w = torch.where(some, torch.softmax(torch.where(some, x, 0.0), -1), 0.0)
                vs = torch.where(seen.any(0)[:, None], vh, 0.0)
                mine = self._weighed(w, seen, vs)
                out[r0 : r0 + n, h] = mine
                size, mine = w @ torch.nan_to_num(vs, nan=0.0, posinf=0.0, neginf=0.0).abs(), mine.abs()
                off = (torch.where(seen, q.abs() @ kh.abs().t(), 0.0).amax(-1, keepdim=True) * abs(scale)
                       * (self.dim + 8) * 2.0**-24)  # fmt: skip
                sub = 2.0**-25 * (vs.abs().sum(0) + (s + n) * mine) if self.dtype == torch.float16 else 0.0
                sub = sub + step * torch.finfo(self.dtype).tiny
                bound[r0 : r0 + n, h] = torch.where(some, (step * mine + step * (size + mine)) * (1 + 2.0**-6)
                                                    + size * (2 * off + (s + n + 16) * 2.0**-23) + sub, 0.0)  # fmt: skip
        return out, bound

    @staticmethod
    def _weighed(w, seen, v):
        """w @ v where a weight of zero at an unseen key takes nothing of its value, whatever that is."""
        if bool(torch.isfinite(v).all()):
            return w @ v
        return torch.where(seen[:, :, None], w[:, :, None] * v[None], 0.0).sum(1)


# ---------------------------------------------------------------------------------------------- sampling
def sampled(logits, uniforms, temperature, top_k=None, top_p=None, min_p=None):
    """The tokens row by row, in float64 on the host; the settings one a row."""
    rows, vocab = logits.shape
    got = torch.empty(rows, dtype=torch.int64)
    for r in range(rows):
        x, t = logits[r].double(), float(temperature[r])
        nan = x.isnan().nonzero()
        if not t > 0 or len(nan) or x.max().abs() == math.inf:
            got[r] = nan[0] if len(nan) else (x == x.max()).nonzero()[0]
            continue
        order = torch.sort(x, descending=True, stable=True).indices
        w = torch.exp((x - x.max()) / t)
        ranked = w[order]
        k = 0 if top_k is None else int(top_k[r])
        left = ranked[:k] if 0 < k < vocab else ranked
        p = 1.0 if top_p is None else float(top_p[r])
        many = left.numel()
        if p < 1:
            before = torch.cumsum(left, 0) - left
            many = max(1, int((before < p * left.sum()).sum()))
        kept = torch.zeros(vocab, dtype=torch.bool).index_fill_(0, order[:many], True)
        low = 0.0 if min_p is None else float(min_p[r])
        if low > 0:
            kept &= w >= min(low, 1.0)
        w = torch.where(kept, w, 0.0)
        cum = w.cumsum(0)
        j = int((cum <= float(uniforms[r]) * float(cum[-1])).sum())
        got[r] = min(j, int(w.nonzero()[-1]))
    return got


# -------------------------------------------------------------------------------------------- acceptance
def accepted(tokens, drafts, parents, cu, max_path):
    """(tokens, path, counts) of accept_tree, node by node."""
    n = len(cu) - 1
    out = torch.full((n, max_path), -1, dtype=torch.int64)
    path = torch.full((n, max_path), -1, dtype=torch.int32)
    counts = torch.zeros(n, dtype=torch.int32)
    for b in range(n):
        lo, hi = int(cu[b]), int(cu[b + 1])
        node = 0 if hi > lo else -1
        while node >= 0 and int(counts[b]) < max_path:
            t = int(tokens[lo + node])
            out[b, counts[b]], path[b, counts[b]] = t, node
            counts[b] += 1
            node = next((i for i in range(node + 1, hi - lo) if int(parents[lo + i]) == node and int(drafts[lo + i]) == t and t >= 0), -1)
    return out, path, counts


def moved(pool, tables, start, path, counts):
    """The pool after the paths' rows have moved together."""
    old, new, bs = pool, pool.clone(), pool.size(4)
    for b in range(len(counts)):
        for j in range(int(counts[b])):
            src, dst = int(start[b]) + int(path[b, j]), int(start[b]) + j
            new[tables[b, dst // bs], :, :, :, dst % bs] = old[tables[b, src // bs], :, :, :, src % bs]
    return new


__all__ = ["LAYER", "Tree", "accepted", "grown", "lines_of", "moved", "packed", "sampled", "unpacked"]
