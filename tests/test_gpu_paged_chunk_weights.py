"""paged_chunk where one key outweighs thousands of others whose values make up the output (a first token that takes the
attention and has no value): weights far below the row's largest keep the type's precision, in float16 too."""

from __future__ import annotations

import math

import pytest
import torch

from tests.chunk_cases import LAYER, Chunk, assert_within, half_step
from tests.test_gpu_paged_chunk import run
from tokquay_amd import ops

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16

# By one workgroup a (sequence, K/V head): keys in parts and not; by shared tiles: in parts, not, and from the queue.
SHAPES = {
    "token_in_parts": [(4000, 1)],
    "tokens": [(1000, 1)] * 130,
    "chunk_in_parts": [(3900, 100)],
    "chunks": [(700, 100)] * 40,
    "chunks_from_the_queue": [(1700, 400)] * 60,
}


def expected(c):
    """(out, bound) float64; the bound on ``|out - kernel|``, in ``Chunk.expected``'s terms (half a step of the output and of each weight; the scores'
    float32 sums), but for float16's subnormal weights: the running maximum is at least 7 powers of two below the largest score
    met so far, so a row's (or a part of a row's) largest weight is at least 2^7, and a weight's subnormal rounding, at most
    2^-25, at most 2^-32 of it."""
    out = torch.zeros(c.q.shape, dtype=torch.float64)
    bound = torch.zeros_like(out)
    group, d = c.heads // c.kv_heads, half_step(c.dtype)
    scale = 1 / math.sqrt(c.dim)
    for b, (s, n) in enumerate(c.seqs):
        k, v = c.keys_values(b)
        r0 = int(c.cu[b])
        unseen = torch.arange(s + n)[None, :] > (s + torch.arange(n))[:, None]
        for h in range(c.heads):
            q, kh, vh = c.q[r0 : r0 + n, h].double(), k[:, h // group], v[:, h // group]
            w = torch.softmax((q @ kh.t() * scale).masked_fill(unseen, -math.inf), -1)
            out[r0 : r0 + n, h] = w @ vh
            size, mine = w @ vh.abs(), out[r0 : r0 + n, h].abs()
            off = (q.abs() @ kh.abs().t()).amax(-1, keepdim=True) * scale * (c.dim + 8) * 2.0**-24
            sub = d * torch.finfo(c.dtype).tiny
            if c.dtype == FP16:
                sub = sub + 2.0**-32 * w.amax(-1, keepdim=True) * (vh.abs().sum(0) + (s + n) * mine)
            bound[r0 : r0 + n, h] = ((d * mine + d * (size + mine)) * (1 + 2.0**-6)
                                     + size * (2 * off + (s + n + 16) * 2.0**-23) + sub)  # fmt: skip
    return out, bound


@pytest.mark.parametrize("nats", [16.0, 17.5])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_keys_far_below_one_without_value(shape, dtype, dim, nats):
    few = shape in ("token_in_parts", "chunk_in_parts")
    c = Chunk(SHAPES[shape], 8 if few else 4, 2 if few else 1, dim, dtype, 16, seed=30)
    c.pool[:, LAYER, 0] = 0
    c.pool[:, LAYER, 1] = c.pool[:, LAYER, 1].clamp(-3, 3) * 4 + 16
    first = c.tables[:, 0].long()
    c.pool[first, LAYER, 0, :, 0] = round(nats / math.sqrt(dim) * 64) / 64
    c.pool[first, LAYER, 1, :, 0] = 0
    c.q[:] = (1 - torch.arange(c.heads) / 64)[:, None]  # heads of 16 or 17.5 nats and somewhat less
    words = ops.chunk_workspace_bytes(len(c.seqs), c.heads, c.kv_heads, dim, c.q.size(0), c.max_new, c.max_context) // 4
    assert (words > 0) == (shape not in ("tokens", "chunks")) and (words % (dim + 2) == 0) == (shape != "chunks_from_the_queue")
    assert_within(run(c), *expected(c))


@pytest.mark.parametrize("seqs", [[(600, 3)], [(600, 200)]])
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_of_tens_of_millions_stay_finite(dim, seqs):
    # Scores come in steps of 2 and 4: how far one lies above the running maximum has to be told from their difference.
    c = Chunk(seqs, 4, 2, dim, FP16, 16, seed=31, garbage=1.0)
    c.pool[:, LAYER, 0] *= 3000
    c.q *= 2000
    out = run(c)
    assert bool(out.isfinite().all())
    k = [c.keys_values(b)[0] for b in range(len(seqs))]
    top = max(float((c.q[:, h].double() @ k[0][:, h // 2].t()).abs().max()) for h in range(4)) / math.sqrt(dim) * 1.4427
    assert 2.0**24 < top < 2.0**27
