"""A run of the three operators as a serving loop uses them: steps of drafted tokens through one attention layer, each
stage against its plain float64 form on what the stage before left, the cache carried from step to step."""

from __future__ import annotations

import math

import pytest
import torch

from tests.chunk_cases import Chunk, assert_within, rotated, rotation_bound, verified
from tokquay_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_steps_of_drafted_tokens(dtype, dim):
    heads, kv_heads, bs, vocab, width = 8, 2, 16, 5003, 256
    gen = torch.Generator().manual_seed(1)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    embed = randn(vocab, width).to(dtype).cuda()
    w_qkv = (randn(width, (heads + 2 * kv_heads) * dim) / math.sqrt(width)).to(dtype).cuda()
    w_out = (randn(heads * dim, vocab) / math.sqrt(heads * dim) * 4).to(dtype).cuda()
    norms = [(torch.rand(dim, generator=gen) + 0.5).to(dtype).cuda() for _ in range(2)]
    table = ops.rope_table(4096, dim).cuda()
    temperature = torch.tensor([1.0, 0.0, 0.8])
    # Prompts already cached: random keys and values.
    start = [700, 33, 2050]
    c = Chunk([(s, 60) for s in start], heads, kv_heads, dim, dtype, bs, seed=2)
    pool, tables = c.pool.cuda(), c.tables.cuda()
    last = torch.randint(0, vocab, (3,), generator=gen)
    emitted = 0
    for step in range(4):
        rows = [5, 4, 1] if step == 2 else [5, 5, 5]
        drafts_of = [torch.randint(0, vocab, (n - 1,), generator=gen) for n in rows]
        cu = [0]
        for n in rows:
            cu.append(cu[-1] + n)
        n = cu[-1]
        ids = torch.cat([torch.cat([last[b : b + 1], drafts_of[b]]) for b in range(3)])
        positions = torch.cat([start[b] + torch.arange(rows[b]) for b in range(3)])
        slots = torch.cat([c.tables[b, (start[b] + torch.arange(rows[b])) // bs].long() * bs
                           + (start[b] + torch.arange(rows[b])) % bs for b in range(3)])  # fmt: skip
        cu_t, start_t = torch.tensor(cu, dtype=torch.int32), torch.tensor(start, dtype=torch.int32)
        qkv = embed[ids.cuda()] @ w_qkv
        q, k, v = (qkv[:, a * dim : b * dim] for a, b in ((0, heads), (heads, heads + kv_heads), (heads + kv_heads, heads + 2 * kv_heads)))
        q_out, out = torch.empty(n, heads, dim, dtype=dtype, device="cuda"), torch.empty(n, heads, dim, dtype=dtype, device="cuda")
        ops.rope_cache_write(q_out, q, k, v, pool, 1, slots.cuda(), positions.cuda(), table, q_norm=norms[0], k_norm=norms[1])
        ops.paged_chunk(out, q_out, pool, 1, tables, cu_t.cuda(), start_t.cuda(), max(rows), max(s + r for s, r in zip(start, rows)))
        logits = (out.view(n, -1) @ w_out).float()
        # A draft model that is right half of the time: the target's best token, or any.
        drafts = torch.zeros(n, dtype=torch.int64)
        best = logits.argmax(-1).cpu()
        for b in range(3):
            for i in range(rows[b] - 1):
                drafts[cu[b] + i] = best[cu[b] + i] if (b + i + step) % 2 else drafts_of[b][i]
        probs = torch.softmax(logits + randn(n, vocab).cuda(), -1)
        uniforms = torch.rand(n, generator=gen)
        tokens, accepted = ops.verify_drafts(logits, drafts.cuda(), uniforms.cuda(), cu_t.cuda(), max(rows),
                                             temperature.cuda(), probs if step % 2 else None)  # fmt: skip

        for got, x, w in ((q_out, q, norms[0]), (pool[slots.cuda() // bs, 1, 0, :, slots.cuda() % bs], k, norms[1])):
            y, size = rotated(x.cpu().view(n, -1, dim), table.cpu(), positions, False, w.cpu(), 1e-6)
            assert_within(got, y, rotation_bound(y, size, dtype))
        assert torch.equal(pool[slots.cuda() // bs, 1, 1, :, slots.cuda() % bs], v.view(n, kv_heads, dim))
        c.seqs, c.cu, c.q, c.pool = [(start[b], rows[b]) for b in range(3)], cu_t, q_out.cpu(), pool.cpu()
        assert_within(out, *c.expected())
        want, count = verified(logits, drafts, uniforms, cu, max(rows), temperature, probs if step % 2 else None)
        assert torch.equal(tokens.cpu(), want) and torch.equal(accepted.cpu(), count)
        emitted += int((want >= 0).sum())
        # Accepted tokens stay in the cache; what was written behind them is overwritten by the next step.
        last = want.gather(1, count.long()[:, None])[:, 0]
        start = [start[b] + int(count[b]) + 1 for b in range(3)]
    assert emitted >= 12
