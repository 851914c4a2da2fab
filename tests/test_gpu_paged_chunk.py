"""paged_chunk against attention in float64: types, head layouts, lengths, block sizes, strides, masked places, errors,
streams and graphs. Tolerances are Chunk.expected's."""

from __future__ import annotations

import math

import pytest
import torch

from tests.chunk_cases import LAYER, Chunk, assert_within
from tokquay_amd import _lib, ops

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def run(c: Chunk, scale=None, q=None, out=None, err=None, pool=None, max_new=None, max_context=None):
    q = c.q.cuda() if q is None else q
    out = torch.full_like(q, 7.0) if out is None else out
    ops.paged_chunk(out, q, c.pool.cuda() if pool is None else pool, LAYER, c.tables.cuda(), c.cu.cuda(), c.start.cuda(),
                    max_new or c.max_new, max_context or c.max_context, scale, d_error=err)  # fmt: skip
    return out


def check(c: Chunk, scale=None, **more):
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = run(c, scale, err=err, **more)
    want, bound = c.expected(scale)
    assert_within(out, want, bound)
    outside = bound.isnan()
    assert bool((out.cpu()[outside] == 7.0).all())  # rows of no sequence are left alone
    assert int(err) == 0


# (start, new) of each sequence: single tokens, drafts, chunks, whole prompts, empty ones.
LENGTHS = {
    "first_token": [(0, 1)],
    "tokens": [(0, 1), (15, 1), (16, 1), (130, 1), (31, 1), (700, 1)],
    "drafts": [(40, 5), (0, 3), (127, 7), (500, 1), (63, 2)],
    "chunks": [(0, 33), (100, 70), (17, 1), (31, 130)],
    "prompts": [(0, 257), (0, 1), (0, 96)],
    "some_empty": [(5, 0), (9, 2), (0, 0), (64, 17), (3, 0)],
}


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", list(LENGTHS))
def test_lengths(lengths, dim, dtype):
    check(Chunk(LENGTHS[lengths], 8, 2, dim, dtype, 16, seed=1, before=2, behind=3))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (12, 12), (7, 1), (6, 2), (16, 2), (20, 1), (40, 2)])
@pytest.mark.parametrize("dim", [64, 128])
def test_head_layouts(heads, kv_heads, dim):
    check(Chunk([(70, 3), (0, 40), (200, 1), (33, 9)], heads, kv_heads, dim, BF16, 16, seed=2))


@pytest.mark.parametrize("block_size", [1, 3, 8, 48, 64, 1024])
@pytest.mark.parametrize("dim", [64, 128])
def test_block_sizes(block_size, dim):
    check(Chunk([(70, 3), (0, 140), (301, 1)], 4, 2, dim, FP16, block_size, seed=3))


@pytest.mark.parametrize("seqs", [[(5000, 1)], [(4095, 4)], [(3000, 150)], [(4100, 1), (0, 5), (900, 1)]])
@pytest.mark.parametrize("dim,dtype", [(64, FP16), (128, BF16)])
def test_long_contexts_in_parts(seqs, dim, dtype):
    c = Chunk(seqs, 8, 2, dim, dtype, 16, seed=4)
    assert ops.chunk_workspace_bytes(len(seqs), 8, 2, dim, c.q.size(0), c.max_new, c.max_context) > 0
    check(c)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (12, 12), (7, 1), (16, 2), (40, 2)])
@pytest.mark.parametrize("dim", [64, 128])
def test_head_layouts_in_parts(heads, kv_heads, dim):
    # 257 positions end a part of 128 or 256 keys one key behind its border.
    c = Chunk([(1200, 3), (2060, 40), (255, 1), (256, 1), (257, 0)], heads, kv_heads, dim, FP16, 16, seed=23)
    assert ops.chunk_workspace_bytes(5, heads, kv_heads, dim, c.q.size(0), c.max_new, c.max_context) > 0
    check(c)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dim", [64, 128])
def test_places_in_parts_that_no_row_sees(dim, bad):
    c = Chunk([(1500, 200), (2100, 3)], 4, 1, dim, BF16, 16, seed=24, garbage=bad)
    assert ops.chunk_workspace_bytes(2, 4, 1, dim, c.q.size(0), c.max_new, c.max_context) > 0
    check(c)


@pytest.mark.parametrize("seqs", [[(0, 256)] * 16, [(300, 1)] * 8, [(0, 1023)] * 2])
def test_short_contexts_stay_in_one_part(seqs):
    c = Chunk(seqs, 12, 12, 64, FP16, 16, seed=25)
    assert ops.chunk_workspace_bytes(len(seqs), 12, 12, 64, c.q.size(0), c.max_new, c.max_context) == 0
    check(c)


@pytest.mark.parametrize("group", [1, 4])
def test_many_rows(group):
    check(Chunk([(300, 500), (0, 1029)], 2 * group, 2, 128, BF16, 16, seed=5))
    check(Chunk([(300, 500), (0, 1029)], 2 * group, 2, 64, FP16, 16, seed=5))


def test_one_sequence_of_many_rows_and_a_long_context():
    check(Chunk([(2500, 300)], 4, 1, 128, BF16, 16, seed=6))


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.5])
def test_scales(scale):
    check(Chunk([(70, 3), (0, 40), (200, 1)], 4, 2, 64, BF16, 16, seed=7), scale=scale)


def test_peaked_scores_raise_the_running_maximum():
    # Keys grow along the sequence, so later tiles exceed the running maximum by far, again and again.
    c = Chunk([(600, 9), (0, 300)], 4, 2, 128, BF16, 16, seed=8, peak=6.0)
    for b in range(2):
        s, n = c.seqs[b]
        for p in range(s + n):
            blk, off = c.slot(b, p)
            c.pool[blk, LAYER, 0, :, off] *= 1 + p / 64
    check(c)


def test_bounds_larger_than_the_lengths():
    c = Chunk([(70, 3), (0, 40), (200, 1)], 4, 2, 64, BF16, 16, seed=9, extra_columns=200)
    check(c, max_new=97, max_context=3000)
    check(c, max_new=40, max_context=3000)
    check(c, max_new=1000, max_context=1000)


@pytest.mark.parametrize("dim", [64, 128])
def test_strided_rows(dim):
    c = Chunk([(70, 3), (0, 40), (200, 1)], 4, 2, dim, BF16, 16, seed=10, before=1)
    rows = c.q.size(0)
    qkv = torch.randn(rows, 8 * dim + 8, dtype=BF16, device="cuda")
    q = qkv[:, 8 : 8 + 4 * dim]
    q.copy_(c.q.view(rows, -1))
    wide = torch.full((rows, 4 * dim + 12), 7.0, dtype=BF16, device="cuda")
    out = wide[:, 4 : 4 + 4 * dim]
    run(c, q=q, out=out)
    want, bound = c.expected()
    assert_within(out.reshape(rows, 4, dim), want, bound)
    assert bool((wide[:, :4] == 7.0).all()) and bool((wide[:, 4 + 4 * dim :] == 7.0).all())
    assert bool((out[0] == 7.0).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("seqs", [[(70, 3), (30, 1)], [(10, 200)], [(3000, 2)], [(45, 9), (0, 70)]])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_a_row_does_not_see_does_not_reach_it(seqs, dim, bad):
    # Unowned slots (also those behind the last key in its block), and the last token's own K and V.
    c = Chunk(seqs, 8, 2, dim, BF16, 16, seed=11, garbage=bad)
    for b, (s, n) in enumerate(seqs):
        if n > 1:
            blk, off = c.slot(b, s + n - 1)
            c.pool[blk, LAYER, :, :, off] = bad
    out = run(c)
    for b, (s, n) in enumerate(seqs):  # the last row sees the bad token: leave it out of the oracle
        if n > 1:
            assert not bool(out[int(c.cu[b + 1]) - 1].isfinite().any())
            blk, off = c.slot(b, s + n - 1)
            c.pool[blk, LAYER, :, :, off] = 0
    want, bound = c.expected()
    for b, (s, n) in enumerate(seqs):
        if n > 1:
            bound[int(c.cu[b + 1]) - 1] = math.nan
    assert_within(out, want, bound)


@pytest.mark.parametrize("dim", [64, 128])
def test_an_infinite_value_reaches_the_rows_that_see_it(dim):
    c = Chunk([(20, 60)], 4, 2, dim, FP16, 16, seed=12)
    blk, off = c.slot(0, 50)
    c.pool[blk, LAYER, 1, :, off, 5] = math.inf
    out = run(c).float().cpu()
    assert bool((out[30:, :, 5] == math.inf).all())  # row 30 is position 50
    assert bool(out[:30].isfinite().all()) and bool(out[:, :, 6:].isfinite().all()) and bool(out[:, :, :5].isfinite().all())


def test_errors_are_flagged_and_stay_in_bounds():
    err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def flags(c, **more):
        err.zero_()
        out = run(c, err=err, **more)
        return int(err), out.cpu()

    def case():
        return Chunk([(70, 3), (0, 40), (200, 1)], 4, 2, 64, BF16, 16, seed=13)

    want, bound = case().expected()
    c = case()
    c.tables[1, 1] = c.pool.size(0)  # past the pool
    got, out = flags(c)
    assert got == _lib.DEVERR_BLOCK_ID
    others = bound.clone()
    others[3:43] = math.nan
    assert_within(out, want, others)
    c = case()
    c.tables[2, 3] = -1
    assert flags(c)[0] == _lib.DEVERR_BLOCK_ID
    for spoil in ({"max_new": 39}, {"max_context": 200}):
        got, out = flags(case(), **spoil)
        assert got == _lib.DEVERR_LENGTH
        lost = slice(3, 43) if "max_new" in spoil else slice(43, 44)
        assert bool((out[lost] == 7.0).all())
        others = bound.clone()
        others[lost] = math.nan
        assert_within(out, want, others)
    c = case()
    c.start[0] = -1
    assert flags(c)[0] == _lib.DEVERR_LENGTH
    c = case()
    c.cu[3] = 60  # rows past q
    assert flags(c)[0] == _lib.DEVERR_LENGTH
    c = case()
    c.start[2] = c.tables.size(1) * 16  # past the table
    assert flags(c, max_context=5000)[0] == _lib.DEVERR_LENGTH


def test_no_rows():
    c = Chunk([(70, 3)], 4, 2, 64, BF16, 16, seed=14)
    pool, tables = c.pool.cuda(), c.tables.cuda()
    empty = torch.empty(0, 4, 64, dtype=BF16, device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.paged_chunk(empty, empty, pool, LAYER, tables[:0], zero, zero[:0], 0, 0)
    ops.paged_chunk(empty, empty, pool, LAYER, tables, torch.zeros(2, dtype=torch.int32, device="cuda"), zero, 0, 0)


def test_a_pool_past_2_31_elements():
    bs, hk, d = 1024, 1, 128
    blocks = 2**31 // (bs * hk * d * 4) + 9  # LAYERS * 2 = 4 slabs a block
    c = Chunk([(1500, 2), (700, 40)], 4, hk, d, BF16, bs, seed=15)
    pool = torch.full((blocks, 2, 2, hk, bs, d), 50.0, dtype=BF16, device="cuda")
    far = blocks - c.pool.size(0)
    pool[far:] = c.pool.cuda()
    want, bound = c.expected()
    c.tables += far
    assert_within(run(c, pool=pool), want, bound)


def test_calls_on_two_streams_at_once():
    a, b = (Chunk([(4000, 3)], 8, 2, 128, BF16, 16, seed=s) for s in (16, 17))
    args = [(c.q.cuda(), c.pool.cuda(), c.tables.cuda(), c.cu.cuda(), c.start.cuda(), torch.empty_like(c.q, device="cuda"))
            for c in (a, b)]  # fmt: skip
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for c, s, (q, pool, tables, cu, start, out) in zip((a, b), streams, args):
            with torch.cuda.stream(s):
                ops.paged_chunk(out, q, pool, LAYER, tables, cu, start, c.max_new, c.max_context)
    torch.cuda.synchronize()
    for c, (*_, out) in zip((a, b), args):
        assert_within(out, *c.expected())


def test_a_captured_call_replays_with_other_lengths():
    small = Chunk([(40, 2), (9, 1)], 8, 2, 64, FP16, 16, seed=18)
    large = Chunk([(2000, 2), (700, 1)], 8, 2, 64, FP16, 16, seed=19)
    blocks = max(small.pool.size(0), large.pool.size(0))
    pool = torch.zeros(blocks, *large.pool.shape[1:], dtype=FP16, device="cuda")
    q, out = torch.zeros_like(large.q, device="cuda"), torch.zeros_like(large.q, device="cuda")
    tables, cu, start = torch.zeros_like(large.tables, device="cuda"), large.cu.cuda(), torch.zeros_like(large.start, device="cuda")

    def put(c):
        pool[: c.pool.size(0)] = c.pool.cuda()
        q.copy_(c.q)
        tables.zero_()
        tables[:, : c.tables.size(1)] = c.tables.cuda()
        start.copy_(c.start)

    def call():
        ops.paged_chunk(out, q, pool, LAYER, tables, cu, start, 2, 2002)

    put(large)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for c in (small, large, small, large):
        put(c)
        out.fill_(7.0)
        graph.replay()
        got = out.clone()
        assert_within(got, *c.expected())
        call()
        assert torch.equal(out, got)


def test_calls_repeat_bit_for_bit():
    c = Chunk([(4000, 3), (100, 70)], 8, 2, 128, BF16, 16, seed=20)
    first = run(c)
    for _ in range(3):
        assert torch.equal(run(c), first)


def test_refusals():
    c = Chunk([(70, 3), (0, 40)], 4, 2, 64, BF16, 16, seed=21)
    good = dict(out=torch.empty_like(c.q, device="cuda"), q=c.q.cuda(), pool=c.pool.cuda(), layer=LAYER,
                block_tables=c.tables.cuda(), cu_seqlens_q=c.cu.cuda(), q_start=c.start.cuda(), max_query_len=40,
                max_context_len=73)  # fmt: skip
    ops.paged_chunk(**good)
    for name, value in [("q", c.q.cuda().half()), ("q", c.q.cuda()[:, :3]), ("out", good["out"][:-1]),
                        ("pool", c.pool.cuda().float()), ("pool", c.pool.cuda()[..., :32].contiguous()), ("layer", 2),
                        ("block_tables", c.tables.cuda().long()), ("cu_seqlens_q", c.cu.cuda()[:-1]),
                        ("q_start", c.start.cuda().long()), ("max_query_len", -1), ("scale", math.inf),
                        ("workspace", torch.empty(8, device="cuda")[::2])]:  # fmt: skip
        with pytest.raises((ValueError, _lib.KernelError), match="paged_chunk"):
            ops.paged_chunk(**{**good, name: value})
    long = Chunk([(3000, 1)], 4, 2, 64, BF16, 16, seed=22)
    with pytest.raises(_lib.KernelError, match="workspace"):
        ops.paged_chunk(torch.empty_like(long.q, device="cuda"), long.q.cuda(), long.pool.cuda(), LAYER,
                        long.tables.cuda(), long.cu.cuda(), long.start.cuda(), 1, 3001,
                        workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))  # fmt: skip


def test_refusals_of_values():
    c = Chunk([(70, 3), (0, 40)], 4, 2, 64, BF16, 16, seed=21)
    good = dict(out=torch.empty_like(c.q, device="cuda"), q=c.q.cuda(), pool=c.pool.cuda(), layer=LAYER,
                block_tables=c.tables.cuda(), cu_seqlens_q=c.cu.cuda(), q_start=c.start.cuda(), max_query_len=40,
                max_context_len=73)  # fmt: skip
    for name, value in [("scale", math.inf), ("scale", math.nan), ("scale", 1e300), ("max_context_len", 2**30 + 1),
                        ("max_context_len", 0), ("max_query_len", 2**30), ("block_tables", c.tables.cuda()[:, :0])]:  # fmt: skip
        with pytest.raises(ValueError, match="paged_chunk"):
            ops.paged_chunk(**{**good, name: value})
    ops.paged_chunk(**{**good, "max_query_len": 0, "max_context_len": 0, "block_tables": c.tables.cuda()[:, :0]})
