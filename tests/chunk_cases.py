"""Inputs and plain float64 forms for the tests of rope_cache_write, paged_chunk and verify_drafts."""

from __future__ import annotations

import math
import random

import torch

from oracle.paged_ref import cdiv

LAYERS, LAYER = 2, 1


def half_step(dtype: torch.dtype) -> float:
    """A rounding to ``dtype`` is off by at most this, relative to the value."""
    return torch.finfo(dtype).eps / 2


# ----------------------------------------------------------------------------------------- rotation
def rotated(x, table, positions, interleaved, weight, eps):
    """Norm (where ``weight``) and rotation of heads ``[N, H, D]`` in float64; also, per element, the sum of
    the magnitudes of what it is made of."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    r = table.size(1)
    y, size = x.clone(), x.abs()
    for i in range(r // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
        c, s = table[positions, i].double()[:, None], table[positions, r // 2 + i].double()[:, None]
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
        size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size


def rotation_bound(y, size, dtype):
    """One rounding to ``dtype`` (half a step of the value; of the smallest normal one below that, where steps stop
    shrinking: half_step * tiny, 2^-25 in float16); float32 inside: the head's sum of squares (its terms are positive: at most 20 roundings
    of 2^-24 relative, halved by the root), root, quotient, two products, then two products and a sum."""
    return half_step(dtype) * y.abs() + 2.0**-24 * 20 * size + half_step(dtype) * torch.finfo(dtype).tiny


# ---------------------------------------------------------------------------------------- attention
class Chunk:
    """A call of paged_chunk: sequences of ``(start, new)`` tokens over a pool whose unowned slots hold ``garbage``."""

    def __init__(self, seqs, heads, kv_heads, dim, dtype, block_size, seed=0, garbage=50.0, before=0, behind=0,
                 extra_columns=1, peak=1.0):  # fmt: skip
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.heads, self.kv_heads, self.dim, self.dtype, self.bs = seqs, heads, kv_heads, dim, dtype, block_size
        need = [cdiv(s + n, block_size) for s, n in seqs]
        blocks = sum(need) + 3
        ids = list(range(blocks))
        random.Random(seed).shuffle(ids)
        pool = torch.full((blocks, LAYERS, 2, kv_heads, block_size, dim), garbage)
        self.tables = torch.zeros(len(seqs), max([1] + need) + extra_columns, dtype=torch.int32)
        for b, (s, n) in enumerate(seqs):
            mine, ids = ids[: need[b]], ids[need[b] :]
            self.tables[b, : len(mine)] = torch.tensor(mine, dtype=torch.int32)
            p = torch.arange(s + n)
            blk = self.tables[b, p // block_size].long()
            pool[blk, LAYER, :, :, p % block_size] = torch.randn(s + n, 2, kv_heads, dim, generator=g)
        self.pool = pool.to(dtype)
        rows = before + sum(n for _, n in seqs) + behind
        self.q = (torch.randn(rows, heads, dim, generator=g) * peak).to(dtype)
        cu = [before]
        for _, n in seqs:
            cu.append(cu[-1] + n)
        self.cu = torch.tensor(cu, dtype=torch.int32)
        self.start = torch.tensor([s for s, _ in seqs], dtype=torch.int32)
        self.max_new = max(n for _, n in seqs)
        self.max_context = max(s + n for s, n in seqs)

    def slot(self, b, position):
        """(block, offset) of a sequence's position."""
        return int(self.tables[b, position // self.bs]), position % self.bs

    def keys_values(self, b):
        s, n = self.seqs[b]
        p = torch.arange(s + n)
        kv = self.pool[self.tables[b, p // self.bs].long(), LAYER, :, :, p % self.bs].double()  # [ctx, 2, Hkv, D]
        return kv[:, 0], kv[:, 1]

    def expected(self, scale=None):
        """(out, bound) float64; rows of no sequence are NaN in both. The bound on ``|out - kernel|``:

        * the output's rounding: half a step of |out| (of the smallest normal value below that);
        * each weight's before it meets V and is summed: with w_j (1 + d_j), |d_j| <= d = half a step, in place of w_j (their sum
          1), sum w (1 + d_j) v / sum w (1 + d_j) - sum w v = sum w d_j (v - out) / sum w (1 + d_j), at most
          d (sum w |v| + |out|) / (1 - d); for weights that are subnormal in float16, 2^-25 of each |v| + |out| instead (the
          largest weight is at least 1);
        * scores: D products summed in float32, off by at most (D + 8) 2^-24 sum |q k| scale, which changes a weight by
          that share; the sum of the weights, and of the products, (keys + 16) 2^-23 more."""
        scale = 1 / math.sqrt(self.dim) if scale is None else scale
        out = torch.full(self.q.shape, math.nan, dtype=torch.float64)
        bound = out.clone()
        group, step = self.heads // self.kv_heads, half_step(self.dtype)
        for b, (s, n) in enumerate(self.seqs):
            if n == 0:
                continue
            k, v = self.keys_values(b)
            r0 = int(self.cu[b])
            unseen = torch.arange(s + n)[None, :] > (s + torch.arange(n))[:, None]
            for h in range(self.heads):
                q, kh = self.q[r0 : r0 + n, h].double(), k[:, h // group]
                vh = v[:, h // group]
                w = torch.softmax((q @ kh.t() * scale).masked_fill(unseen, -math.inf), -1)
                out[r0 : r0 + n, h] = w @ vh
                size = w @ vh.abs()
                off = ((q.abs() @ kh.abs().t()).masked_fill(unseen, 0).amax(-1, keepdim=True) * abs(scale)
                       * (self.dim + 8) * 2.0**-24)  # fmt: skip
                mine = out[r0 : r0 + n, h].abs()
                sub = 2.0**-25 * (vh.abs().sum(0) + (s + n) * mine) if self.dtype == torch.float16 else 0.0
                sub = sub + step * torch.finfo(self.dtype).tiny
                bound[r0 : r0 + n, h] = ((step * mine + step * (size + mine)) * (1 + 2.0**-6)
                                         + size * (2 * off + (s + n + 16) * 2.0**-23) + sub)  # fmt: skip
        return out, bound


def assert_within(got, want, bound):
    """Rows that the oracle has none of (NaN bound) are not looked at."""
    got = got.double().cpu()
    real = ~bound.isnan()
    off = ((got - want).abs() - bound)[real]
    assert bool((off <= 0).all()), f"{int((~(off <= 0)).sum())} of {off.numel()} values off, by up to {float(off.max()):.3g}"


# --------------------------------------------------------------------------------------------- drafts
def verified(logits, drafts, uniforms, cu, max_rows, temperature, probs):
    """The accept / resample rule, sequence by sequence, in float64 on the host."""
    logits, uniforms = logits.cpu(), uniforms.cpu().double()
    tokens = torch.full((len(temperature), max_rows), -1, dtype=torch.int64)
    accepted = torch.zeros(len(temperature), dtype=torch.int32)
    vocab = logits.size(1)

    def one_hot(j):
        return torch.zeros(vocab, dtype=torch.float64).index_fill_(0, torch.tensor([j]), 1.0)

    def argmax(x):  # NaN above every number, then the lowest column
        nan = x.isnan().nonzero()
        return int(nan[0]) if len(nan) else int((x == x.max()).nonzero()[0])

    for b, t in enumerate(float(t) for t in temperature):
        lo, last = int(cu[b]), int(cu[b + 1]) - 1
        if last < lo:
            continue

        def target(row):
            x = logits[row].double()
            if not t > 0 or x.isnan().any() or x.max() == math.inf or x.max() == -math.inf:
                return one_hot(argmax(x))
            return torch.softmax(x / t, -1)

        i = 0
        while lo + i < last:
            p, x = target(lo + i), int(drafts[lo + i])
            q = (one_hot(x) if 0 <= x < vocab else torch.zeros(vocab).double()) if probs is None else probs[lo + i].double().cpu()
            if not (0 <= x < vocab and float(uniforms[lo + i] * q[x]) < float(p[x])):
                rest = torch.clamp(p - q, min=0)
                w = rest if rest.sum() > 0 else p
                break
            tokens[b, i] = x
            i += 1
        else:
            w = target(last)
        cum = w.cumsum(0)
        j = int((cum <= uniforms[last] * cum[-1]).sum())
        tokens[b, i] = min(j, int(w.nonzero()[-1]))
        accepted[b] = i
    return tokens, accepted
