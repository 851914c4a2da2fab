"""paged_tree against attention in float64: types, head layouts, trees, lengths, block sizes, masked places, errors, streams
and graphs. Tolerances are Tree.expected's."""

from __future__ import annotations

import math

import pytest
import torch

from tests.chunk_cases import assert_within
from tests.tree_cases import LAYER, Tree, grown
from tokquay_amd import _lib, ops

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def run(c: Tree, scale=None, q=None, out=None, err=None, pool=None, masks=None, max_new=None, max_context=None):
    q = c.q.cuda() if q is None else q
    out = torch.full_like(q, 7.0) if out is None else out
    ops.paged_tree(out, q, c.pool.cuda() if pool is None else pool, LAYER, c.tables.cuda(), c.cu.cuda(), c.start.cuda(),
                   c.masks.cuda() if masks is None else masks, max_new or c.max_new, max_context or c.max_context, scale,
                   d_error=err)  # fmt: skip
    return out


def check(c: Tree, scale=None, **more):
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = run(c, scale, err=err, **more)
    want, bound = c.expected(scale)
    assert_within(out, want, bound)
    outside = bound.isnan().all(-1).all(-1)
    assert bool((out.cpu()[outside] == 7.0).all())  # rows of no sequence are left alone
    assert int(err) == 0


def trees(*lengths, roots=1):
    return [(s, grown(n, s + n, roots=min(n, roots))) for s, n in lengths]


# (start, nodes) of each sequence.
LENGTHS = {
    "one_node": [(0, 1), (130, 1)],
    "small": [(40, 5), (0, 3), (127, 7), (500, 1), (63, 12)],
    "words": [(0, 33), (100, 70), (17, 1), (31, 130), (64, 64)],
    "some_empty": [(5, 0), (9, 22), (0, 0), (64, 17), (3, 0)],
}


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", list(LENGTHS))
def test_trees(lengths, dim, dtype):
    check(Tree(trees(*LENGTHS[lengths]), 8, 2, dim, dtype, 16, seed=1, before=2, behind=3))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (12, 12), (7, 1), (6, 2), (16, 2), (20, 1), (40, 2)])
@pytest.mark.parametrize("dim", [64, 128])
def test_head_layouts(heads, kv_heads, dim):
    check(Tree(trees((70, 3), (0, 40), (200, 1), (33, 9)), heads, kv_heads, dim, BF16, 16, seed=2))


@pytest.mark.parametrize("block_size", [1, 3, 8, 48, 64, 1024])
@pytest.mark.parametrize("dim", [64, 128])
def test_block_sizes(block_size, dim):
    check(Tree(trees((70, 3), (0, 90), (301, 14)), 4, 2, dim, FP16, block_size, seed=3))


@pytest.mark.parametrize("start", [0, 1, 31, 32, 33, 63, 64, 65, 95])
@pytest.mark.parametrize("nodes", [9, 80])
def test_where_the_tree_begins_in_a_tile(start, nodes):
    check(Tree(trees((start, nodes)), 4, 1, 64, BF16, 16, seed=4))


@pytest.mark.parametrize("group", [1, 2, 3, 4, 7, 8])
def test_row_counts_a_kv_head(group):
    # 9 to 192 rows a K/V head: every kernel.
    for nodes in (9, 15, 24):
        check(Tree(trees((200, nodes), (90, nodes - 3)), group, 1, 128, FP16, 16, seed=5))


@pytest.mark.parametrize("lengths", [[(5000, 1)], [(4095, 14)], [(3000, 150)], [(4100, 20), (0, 5), (900, 1)]])
@pytest.mark.parametrize("dim,dtype", [(64, FP16), (128, BF16)])
def test_long_contexts_in_parts(lengths, dim, dtype):
    c = Tree(trees(*lengths), 8, 2, dim, dtype, 16, seed=6)
    assert ops.tree_workspace_bytes(len(lengths), 8, 2, dim, c.q.size(0), c.max_new, c.max_context) > 0
    check(c)


def test_parts_of_which_a_row_sees_nothing():
    # Every node a root: the 600 rows see a short context and, each in its own part, themselves.
    c = Tree([(100, [-1] * 600)], 1, 1, 64, BF16, 16, seed=7)
    assert ops.tree_workspace_bytes(1, 1, 1, 64, 600, 600, 700) > 0
    check(c)
    check(Tree([(0, [-1] * 600)], 1, 1, 64, FP16, 16, seed=7))


def test_from_the_queue():
    c = Tree(trees(*[(2100 + 3 * i, 33 + i // 2) for i in range(36)]), 32, 8, 128, BF16, 16, seed=8)
    plan = ops.tree_workspace_bytes(36, 32, 8, 128, c.q.size(0), c.max_new, c.max_context)
    assert 0 < plan < 1 << 16  # a queue of row tiles, no sums of parts
    check(c)


def test_large_trees():
    check(Tree([(300, grown(500, 1)), (0, grown(700, 2, roots=3)), (64, grown(300, 3, line=True))], 4, 2, 128, BF16, 16, seed=9))


def test_forests():
    check(Tree(trees((40, 30), (0, 70), roots=6), 4, 2, 64, BF16, 16, seed=10))


def test_masks_of_any_bits():
    # Bits of nodes behind the row's own, of other sequences' numbers, gaps: what lies behind the row is not seen.
    for start, nodes in ((37, 70), (0, 70), (64, 20)):
        c = Tree([(start, grown(nodes, 1)), (5, grown(9, 2))], 4, 2, 64, BF16, 16, seed=11, words=3)
        g = torch.Generator().manual_seed(start)
        c.masks = torch.randint(-(2**63), 2**63 - 1, c.masks.shape, generator=g)
        check(c)


def test_rows_that_see_nothing_are_zero():
    c = Tree([(0, grown(70, 1)), (0, grown(9, 2)), (50, grown(7, 3))], 4, 2, 64, BF16, 16, seed=12, garbage=math.nan)
    c.masks[::3] = 0
    c.masks[71] = 1 << 40  # behind the row
    check(c)
    out = run(c).cpu()
    assert bool((out[:79:3] == 0).all()) and bool((out[71] == 0).all())
    assert bool((out[81] != 0).any())  # cached keys are seen without bits
    # In parts too.
    c = Tree([(0, [-1] * 600)], 1, 1, 64, FP16, 16, seed=13)
    c.masks[5::7] = 0
    check(c)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 6e4])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nodes", [9, 90])
def test_keys_and_values_that_a_row_does_not_see(dim, bad, nodes):
    # Node 3 holds nothing usable; its descendants (none here: it is a leaf) are the only ones to see it.
    parents = [p if p != 3 else 2 for p in grown(nodes, 4)]
    c = Tree([(61, parents), (200, grown(5, 5))], 8, 2, dim, BF16, 16, seed=14, garbage=bad)
    blk, off = c.slot(0, 61 + 3)
    c.pool[blk, LAYER, :, :, off] = bad
    want, bound = c.expected()
    want[3], bound[3] = math.nan, math.nan  # row 3 itself
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert_within(run(c, err=err), want, bound)
    assert int(err) == 0


def test_values_that_some_rows_see():
    # An infinite value in node 2 reaches that node's descendants, and no other row.
    for nodes in (9, 90):
        parents = grown(nodes, 6)
        c = Tree([(61, parents)], 4, 2, 64, BF16, 16, seed=15)
        blk, off = c.slot(0, 63)
        c.pool[blk, LAYER, 1, :, off, 5] = math.inf
        out = run(c).cpu()
        seen = c.seen(0)[:, 63]
        assert bool((out[seen][:, :, 5] == math.inf).all())
        want, bound = c.expected()
        bound[seen, :, 5] = math.nan
        assert_within(out, want, bound)


def test_a_line_is_paged_chunk():
    c = Tree([(100, grown(20, 0, line=True)), (0, grown(70, 0, line=True))], 8, 2, 128, BF16, 16, seed=16)
    out = run(c)
    same = torch.full_like(out, 7.0)
    ops.paged_chunk(same, c.q.cuda(), c.pool.cuda(), LAYER, c.tables.cuda(), c.cu.cuda(), c.start.cuda(), c.max_new, c.max_context)
    assert torch.equal(out, same)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.5])
def test_scales(scale):
    check(Tree(trees((70, 3), (0, 40), (200, 11)), 4, 2, 64, BF16, 16, seed=17), scale=scale)


def test_bounds_larger_than_the_lengths():
    c = Tree(trees((70, 3), (0, 40), (200, 11)), 4, 2, 64, BF16, 16, seed=18, extra_columns=200, words=4)
    check(c, max_new=97, max_context=3000)
    check(c, max_new=256, max_context=1000)


def test_strided_rows():
    c = Tree(trees((70, 30), (0, 40)), 4, 2, 64, BF16, 16, seed=19)
    q = torch.zeros(70, 8 * 64, dtype=BF16, device="cuda")[:, 128:384].view(70, 4, 64)
    q.copy_(c.q)
    out = torch.full((70, 300), 7.0, dtype=BF16, device="cuda")[:, 4:260]
    run(c, q=q, out=out)
    assert_within(out.view(70, 4, 64), *c.expected())


def test_errors_are_flagged_and_other_sequences_right():
    c = Tree(trees((70, 30), (0, 40), (33, 9)), 4, 2, 64, BF16, 16, seed=20)
    want, bound = c.expected()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = run(c, err=err, max_new=39, max_context=c.max_context)
    assert int(err) == _lib.DEVERR_LENGTH
    assert bool((out[30:70] == 7.0).all())
    bound[30:70] = math.nan
    assert_within(out, want, bound)
    err.zero_()
    c.tables[1, 1] = c.pool.size(0)
    out = run(c, err=err)
    assert int(err) == _lib.DEVERR_BLOCK_ID
    assert_within(out, want, bound)


def test_other_streams_and_graphs():
    c = Tree(trees((700, 30), (0, 70), (2000, 12)), 8, 2, 64, BF16, 16, seed=21)
    q, pool, masks = c.q.cuda(), c.pool.cuda(), c.masks.cuda()
    tables, cu, start = c.tables.cuda(), c.cu.cuda(), c.start.cuda()
    args = (pool, LAYER, tables, cu, start, masks, 70, 4000)
    want = torch.empty_like(q)
    ops.paged_tree(want, q, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = torch.empty_like(q)
        ops.paged_tree(out, q, *args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)
    graphs, outs = [], []
    for _ in range(2):  # each with a workspace of its own
        out, graph = torch.zeros_like(q), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_tree(out, q, *args)
        graphs.append(graph)
        outs.append(out)
    for turn in range(3):
        q.copy_(torch.randn(c.q.shape, generator=torch.Generator().manual_seed(turn)).to(BF16))
        masks.copy_(torch.cat([Tree(trees((700, 30), (0, 70), (2000, 12), roots=1 + turn), 8, 2, 64, BF16, 16).masks]))
        for graph in graphs:
            graph.replay()
        ops.paged_tree(want, q, *args)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_offsets_past_2_to_the_31():
    # A pool of 2^32 elements and more, the sequence's blocks at its end.
    c = Tree(trees((300, 20)), 8, 8, 128, BF16, 16, seed=22)
    blocks = 2**31 // (2 * 2 * 8 * 16 * 128) * 2 + 40
    pool = torch.zeros(blocks, 2, 2, 8, 16, 128, dtype=BF16, device="cuda")
    shift = blocks - c.pool.size(0)
    pool[shift:] = c.pool.cuda()
    want, bound = c.expected()
    c.tables += shift
    assert_within(run(c, pool=pool), want, bound)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("start,nodes", [(0, 9), (0, 90), (0, 600), (5, 9), (70, 90)])
def test_rows_whose_scores_are_all_minus_infinity_have_no_softmax(start, nodes, dim):
    # Not the same as a row that sees nothing: NaN, as in a line by paged_chunk.
    c = Tree([(start, grown(nodes, 0, line=True))], 2, 1, dim, BF16, 16, seed=23)
    c.q = c.q.abs().clamp_min(0.25)
    c.pool[:, :, 0, :, :, 0] = -math.inf
    out, same = run(c), torch.empty_like(c.q).cuda()
    ops.paged_chunk(same, c.q.cuda(), c.pool.cuda(), LAYER, c.tables.cuda(), c.cu.cuda(), c.start.cuda(), c.max_new, c.max_context)
    assert bool(same.isnan().all()) and bool(out.isnan().all())
    c.masks[1::3] = 0
    out = run(c)
    blind = torch.arange(nodes) % 3 == 1 if start == 0 else torch.zeros(nodes, dtype=torch.bool)
    assert bool((out[blind] == 0).all()) and bool(out[~blind].isnan().all())
