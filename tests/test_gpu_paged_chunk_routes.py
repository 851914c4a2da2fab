"""paged_chunk over the forms that only larger calls take: row tiles from the queue, and 33 to 64 rows a K/V head. Each test
asserts the form through the workspace's size. Tolerances are Chunk.expected's."""

from __future__ import annotations

import math
import random

import pytest
import torch

from tests.chunk_cases import LAYER, Chunk, assert_within
from tests.test_gpu_paged_chunk import check, run
from tokquay_amd import _lib, ops

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16

QUEUE_WORDS, TILE_ROWS = 288, 128  # in front of the queue's pairs; rows of a pair's tile


def ragged(seed, sequences=40, context=2100):
    """Chunks of 0 to 300 tokens, the longest context ``context``: one of the largest, empty ones among them."""
    rng = random.Random(seed)
    new = [300, 0, 1, 0, 32, 33] + [rng.randint(0, 300) for _ in range(sequences - 6)]
    start = [context - 300, 7, 900, 0, 64, 31] + [rng.choice([0, rng.randint(0, 700)]) for _ in range(sequences - 6)]
    seqs = list(zip(start, new))
    rng.shuffle(seqs)
    return seqs


def workspace(c, max_new=None, max_context=None):
    return ops.chunk_workspace_bytes(len(c.seqs), c.heads, c.kv_heads, c.dim, c.q.size(0), max_new or c.max_new,
                                     max_context or c.max_context)  # fmt: skip


def queued(c, **more):
    pairs = c.q.size(0) * (c.heads // c.kv_heads) // TILE_ROWS + len(c.seqs)
    return workspace(c, **more) == 4 * (QUEUE_WORDS + 2 * pairs)


@pytest.mark.parametrize("heads,kv_heads", [(12, 3), (8, 8), (14, 2)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
def test_ragged_chunks_from_the_queue(dim, dtype, heads, kv_heads):
    c = Chunk(ragged(1, 60), heads, kv_heads, dim, dtype, 16, seed=1, before=2, behind=3)
    assert queued(c)
    check(c)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dim", [64, 128])
def test_places_of_the_queue_that_no_row_sees(dim, bad):
    c = Chunk(ragged(2), 12, 3, dim, BF16, 16, seed=2, garbage=bad)
    assert queued(c)
    check(c)


@pytest.mark.parametrize("dim", [64, 128])
def test_an_infinite_value_in_the_queue_reaches_the_rows_that_see_it(dim):
    c = Chunk(ragged(3), 12, 3, dim, FP16, 16, seed=3)
    assert queued(c)
    want, bound = c.expected()
    b = next(i for i, (s, n) in enumerate(c.seqs) if n >= 200)
    s, n = c.seqs[b]
    blk, off = c.slot(b, s + 150)
    c.pool[blk, LAYER, 1, :, off, 5] = math.inf
    out = run(c).cpu()
    seen = slice(int(c.cu[b]) + 150, int(c.cu[b + 1]))
    assert bool((out[seen, :, 5] == math.inf).all())
    bound[seen, :, 5] = math.nan
    assert_within(out, want, bound)


def test_a_sequence_of_the_queue_that_does_not_fit():
    for spoil in ("new", "context", "start", "table"):
        c = Chunk(ragged(4), 12, 3, 64, BF16, 16, seed=4)
        want, bound = c.expected()
        new, context = c.max_new, c.max_context
        first = max(range(len(c.seqs)), key=lambda b: c.seqs[b])  # the longest: 300 tokens to 2,100
        lost, got = first, _lib.DEVERR_LENGTH
        if spoil == "new":
            new = 299
            assert sorted(n for _, n in c.seqs)[-2] < 300
        elif spoil == "context":
            context = 2099
        elif spoil == "start":
            c.start[lost] = -1
        else:
            c.tables[lost, 3] = c.pool.size(0)
            got = _lib.DEVERR_BLOCK_ID
        assert queued(c, max_new=new, max_context=context)
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = run(c, err=err, max_new=new, max_context=context).cpu()
        assert int(err) == got
        rows = slice(int(c.cu[lost]), int(c.cu[lost + 1]))
        assert spoil == "table" or bool((out[rows] == 7.0).all())
        bound[rows] = math.nan
        assert_within(out, want, bound)


def test_more_row_tiles_than_rows_are_flagged():
    # Offsets that fall and rise again name the same rows many times over: more tiles than the queue has room for.
    c = Chunk([(1800, 300)] + [(0, 0)] * 39, 12, 3, 64, BF16, 16, seed=5)
    assert queued(c)
    c.cu[2::2] = 0
    c.start[2::2] = 1800
    c.tables[2::2] = c.tables[0].clone()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    run(c, err=err)
    assert int(err) == _lib.DEVERR_LENGTH


def test_a_captured_call_of_the_queue_replays_with_other_lengths():
    rows, sequences = 40 * 300, 40
    a, b = (Chunk(ragged(s), 12, 3, 64, FP16, 16, seed=s) for s in (6, 7))
    for c in (a, b):  # rows behind the last sequence up to the captured count
        c.q = torch.cat([c.q, torch.zeros(rows - c.q.size(0), 12, 64, dtype=FP16)])
    blocks, columns = (max(x.pool.size(0) for x in (a, b)), max(x.tables.size(1) for x in (a, b)))
    pool = torch.zeros(blocks, *a.pool.shape[1:], dtype=FP16, device="cuda")
    q, out = torch.zeros_like(a.q, device="cuda"), torch.zeros_like(a.q, device="cuda")
    tables = torch.zeros(sequences, columns, dtype=torch.int32, device="cuda")
    cu, start = torch.zeros_like(a.cu, device="cuda"), torch.zeros_like(a.start, device="cuda")

    def put(c):
        pool[: c.pool.size(0)] = c.pool.cuda()
        q.copy_(c.q)
        tables.zero_()
        tables[:, : c.tables.size(1)] = c.tables.cuda()
        cu.copy_(c.cu)
        start.copy_(c.start)

    def call():
        ops.paged_chunk(out, q, pool, LAYER, tables, cu, start, 300, 2100)

    assert queued(a) and queued(b)
    put(a)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    wants = [c.expected() for c in (a, b)]
    for i in (1, 0, 1, 0):
        put((a, b)[i])
        out.fill_(7.0)
        graph.replay()
        got = out.clone()
        assert_within(got, *wants[i])
        assert bool((got.cpu()[wants[i][1].isnan()] == 7.0).all())
        call()
        assert torch.equal(out, got)


def test_the_queue_repeats_bit_for_bit():
    c = Chunk(ragged(8), 12, 3, 128, BF16, 16, seed=8)
    assert queued(c)
    first = run(c)
    for _ in range(3):
        assert torch.equal(run(c), first)


@pytest.mark.parametrize("heads,kv_heads,new", [(5, 1, 8), (1, 1, 48), (8, 8, 49), (14, 2, 8), (14, 2, 9), (64, 1, 1), (1, 1, 64), (1, 1, 65)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
def test_33_to_65_rows_of_a_head(dim, dtype, heads, kv_heads, new):
    check(Chunk([(300, new), (0, new), (17, 1), (5, 0), (63, max(new - 1, 1))], heads, kv_heads, dim, dtype, 16, seed=9))
    c = Chunk([(4000, new), (1025, 1)], heads, kv_heads, dim, dtype, 16, seed=10)  # in parts
    assert workspace(c) > 0 and workspace(c) % ((dim + 2) * 4 * heads) == 0
    check(c)
