"""A run of the tree operators as a serving loop uses them: steps of drafted trees through one attention layer, each stage against its
plain form on what the stage before left, the cache carried from step to step; and a request forked in between."""

from __future__ import annotations

import math

import pytest
import torch

from tests.chunk_cases import assert_within, rotated, rotation_bound
from tests.tree_cases import Tree, accepted, grown, lines_of, moved, packed, sampled
from tokquay_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_steps_of_drafted_trees(dtype, dim):
    heads, kv_heads, bs, vocab, width, layer = 8, 2, 16, 5003, 256, 1
    gen = torch.Generator().manual_seed(1)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    embed = randn(vocab, width).to(dtype).cuda()
    w_qkv = (randn(width, (heads + 2 * kv_heads) * dim) / math.sqrt(width)).to(dtype).cuda()
    w_out = (randn(heads * dim, vocab) / math.sqrt(heads * dim) * 6).to(dtype).cuda()
    table = ops.rope_table(4096, dim).cuda()
    settings = (torch.tensor([1.0, 0.0, 0.8]), i32([0, 0, 40]), torch.tensor([0.9, 1.0, 0.95]), torch.tensor([0.0, 0.0, 0.02]))
    # Prompts already cached: random keys and values.
    start = [700, 33, 2050]
    c = Tree([(s, grown(160, 1)) for s in start], heads, kv_heads, dim, dtype, bs, seed=2)
    pool, tables = c.pool.cuda(), c.tables.cuda()
    last = torch.randint(0, vocab, (3,), generator=gen)
    emitted = 0
    for step in range(4):
        sizes = [12, 9, 1] if step == 2 else [26, 33, 70]
        trees = [grown(n, 10 * step + n) for n in sizes]
        cu = [0]
        for n in sizes:
            cu.append(cu[-1] + n)
        n, max_new, max_context = cu[-1], max(sizes), max(s + k for s, k in zip(start, sizes))
        drafts = torch.randint(0, vocab, (n,), generator=gen)
        for b in range(3):
            drafts[cu[b]] = last[b]
        cu_t, start_t, parents = i32(cu).cuda(), i32(start).cuda(), i32(sum(trees, [])).cuda()
        positions, masks = ops.tree_layout(parents, cu_t, start_t, max_new)
        slots = torch.cat([c.tables[b, (start[b] + torch.arange(sizes[b])) // bs].long() * bs
                           + (start[b] + torch.arange(sizes[b])) % bs for b in range(3)]).cuda()  # fmt: skip
        qkv = embed[drafts.cuda()] @ w_qkv
        q, k, v = (qkv[:, a * dim : b * dim] for a, b in ((0, heads), (heads, heads + kv_heads), (heads + kv_heads, heads + 2 * kv_heads)))
        q_out, out = torch.empty(n, heads, dim, dtype=dtype, device="cuda"), torch.empty(n, heads, dim, dtype=dtype, device="cuda")
        ops.rope_cache_write(q_out, q, k, v, pool, layer, slots, positions, table)
        ops.paged_tree(out, q_out, pool, layer, tables, cu_t, start_t, masks, max_new, max_context)
        logits = (out.view(n, -1) @ w_out).float()
        uniforms = torch.rand(n, generator=gen)
        tokens = ops.sample_tokens(logits, uniforms.cuda(), *(x.cuda() for x in settings), cu_seqlens_q=cu_t)
        # A draft model that is right for most nodes' first children (drafts were fed before: as if it had known).
        right = drafts.clone()
        for b in range(3):
            for i in range(sizes[b] - 1, 0, -1):
                if (i + step) % 4:
                    right[cu[b] + i] = tokens[cu[b] + trees[b][i]]
        before = pool.cpu()
        got, path, counts = ops.accept_tree(tokens, right.cuda(), parents, cu_t, 20, pool, tables, start_t)

        lines = [x for t in trees for x in lines_of(t)]
        owner = torch.repeat_interleave(torch.arange(3), torch.tensor(sizes))
        assert torch.equal(positions.cpu(), torch.tensor([start[int(b)] + len(x) - 1 for b, x in zip(owner, lines)]))
        assert torch.equal(masks.cpu(), packed(lines, -(-max_new // 64)))
        for x, y in ((q, q_out.cpu()), (k, before[slots.cpu() // bs, layer, 0, :, slots.cpu() % bs])):
            want, size = rotated(x.cpu().view(n, -1, dim), table.cpu(), positions.cpu(), False, None, 1e-6)
            assert_within(y, want, rotation_bound(want, size, dtype))
        c.seqs, c.cu, c.q, c.pool, c.masks = list(zip(start, sizes)), i32(cu), q_out.cpu(), before, masks.cpu()
        assert_within(out, *c.expected())
        assert torch.equal(tokens.cpu(), sampled(logits.cpu(), uniforms, *(x[owner] for x in settings)))
        want = accepted(tokens.cpu(), right, parents.cpu(), cu, 20)
        for g, w in zip((got, path, counts), want):
            assert torch.equal(g.cpu(), w)
        assert torch.equal(pool.cpu(), moved(before, c.tables, start, want[1], want[2]))
        emitted += int(want[2].sum())
        last = want[0].gather(1, want[2].long()[:, None] - 1)[:, 0]
        start = [start[b] + int(want[2][b]) for b in range(3)]
        if step == 1:  # the last sequence goes on from a copy of the first's cache: its whole blocks shared, the filled part of the next copied
            full = start[0] // bs
            ops.copy_blocks(pool, tables[0, full : full + 1].contiguous(), tables[2, full : full + 1].contiguous(), i32([start[0] % bs]).cuda())
            tables[2, :full] = tables[0, :full]
            c.tables = tables.cpu()
            start[2], last[2] = start[0], last[0]
    assert emitted >= 16


def test_a_captured_step_is_replayed_on_other_trees():
    """The whole step in one graph: other trees, lengths, starts and settings from replay to replay, rows behind the last sequence."""
    heads, kv_heads, dim, bs, vocab, rows, max_new, max_context, layer = 8, 2, 64, 16, 5003, 96, 40, 2100, 1
    gen = torch.Generator().manual_seed(5)
    c = Tree([(s, grown(40, 1)) for s in (2060, 100, 700)], heads, kv_heads, dim, torch.bfloat16, bs, seed=6)
    tables, table = c.tables.cuda(), ops.rope_table(4096, dim).cuda()
    buffers = dict(parents=torch.zeros(rows, dtype=torch.int32), cu=torch.zeros(4, dtype=torch.int32),
                   start=torch.zeros(3, dtype=torch.int32), slots=torch.full((rows,), -1), drafts=torch.zeros(rows, dtype=torch.int64),
                   q=torch.zeros(rows, heads * dim, dtype=torch.bfloat16), k=torch.zeros(rows, kv_heads * dim, dtype=torch.bfloat16),
                   v=torch.zeros(rows, kv_heads * dim, dtype=torch.bfloat16), logits=torch.zeros(rows, vocab), uniforms=torch.zeros(rows),
                   temperature=torch.ones(3), top_k=torch.zeros(3, dtype=torch.int32), top_p=torch.ones(3), min_p=torch.zeros(3),
                   pool=c.pool)  # fmt: skip
    buffers = {name: x.cuda() for name, x in buffers.items()}
    error = torch.zeros(1, dtype=torch.int32, device="cuda")

    def step(parents, cu, start, slots, drafts, q, k, v, logits, uniforms, temperature, top_k, top_p, min_p, pool):
        positions, masks = ops.tree_layout(parents, cu, start, max_new, error)
        q_out, out = torch.zeros(rows, heads, dim, dtype=q.dtype, device="cuda"), torch.zeros(rows, heads, dim, dtype=q.dtype, device="cuda")
        ops.rope_cache_write(q_out, q, k, v, pool, layer, slots, positions, table, d_error=error)
        ops.paged_tree(out, q_out, pool, layer, tables, cu, start, masks, max_new, max_context, d_error=error)
        tokens = ops.sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p, cu, error)
        return positions, masks, out, tokens, *ops.accept_tree(tokens, drafts, parents, cu, 12, pool, tables, start, error)

    def refill(turn):
        sizes, start = ([26, 1, 33], [40, 7, 40], [1, 1, 1], [0, 40, 13])[turn], ([2060, 33, 600], [0, 100, 700], [5, 0, 1], [7, 90, 650])[turn]
        cu = [0, sizes[0], sizes[0] + sizes[1], sum(sizes)]
        trees = [grown(n, 7 * turn + b) if n else [] for b, n in enumerate(sizes)]
        slots, logits, drafts = torch.full((rows,), -1), torch.randn(rows, vocab, generator=gen) * 3, torch.randint(0, vocab, (rows,), generator=gen)
        for b in range(3):
            at = start[b] + torch.arange(sizes[b])
            slots[cu[b] : cu[b + 1]] = c.tables[b, at // bs].long() * bs + at % bs
            for i in range(1, sizes[b]):  # greedy rows take the path of first children
                logits[cu[b] + trees[b][i], drafts[cu[b] + i]] = 40.0 - i / 4
        new = dict(parents=torch.tensor(sum(trees, []) + [-1] * (rows - sum(sizes))), cu=torch.tensor(cu), start=torch.tensor(start),
                   slots=slots, drafts=drafts, logits=logits, uniforms=torch.rand(rows, generator=gen), temperature=torch.tensor([0.0, 0.7, 1.0]),
                   top_k=torch.tensor([0, 50, 0]), top_p=torch.tensor([1.0, 0.9, 0.8]), min_p=torch.tensor([0.0, 0.01, 0.0]),
                   pool=c.pool)  # fmt: skip
        for name in ("q", "k", "v"):
            new[name] = torch.randn(buffers[name].shape, generator=gen)
        for name, x in new.items():
            buffers[name].copy_(x)
        return sum(sizes)

    refill(0)
    step(**buffers)  # libraries and allocations are there before the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(**buffers)
    accepts = 0
    for turn in range(4):
        n = refill(turn)
        pool = buffers["pool"].clone()
        want = step(**{**buffers, "pool": pool})
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, expected in zip(captured, want):
            assert torch.equal(got, expected)
        assert torch.equal(buffers["pool"], pool)
        positions, masks, out, tokens, _, _, counts = captured
        assert not positions[n:].any() and not masks[n:].any() and not out[n:].any() and (tokens[n:] == -1).all()
        accepts += int(counts.sum())
    assert accepts > 12 and not error.item()
