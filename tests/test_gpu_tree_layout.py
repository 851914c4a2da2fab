"""tree_layout against the plain definition: whole numbers, equal."""

from __future__ import annotations

import pytest
import torch

from tests.tree_cases import grown, lines_of, packed
from tokquay_amd import _lib, ops

pytestmark = pytest.mark.gpu


def check(trees, starts, before=0, behind=0, max_new=None, words=None):
    max_new = max_new or max([1] + [len(t) for t in trees])
    words = words or -(-max_new // 64)
    cu = [before]
    for t in trees:
        cu.append(cu[-1] + len(t))
    n = cu[-1] + behind
    parents = torch.full((n,), 77, dtype=torch.int32)
    want_p, want_m = torch.zeros(n, dtype=torch.int64), torch.zeros(n, words, dtype=torch.int64)
    for b, t in enumerate(trees):
        if t:
            parents[cu[b] : cu[b + 1]] = torch.tensor(t, dtype=torch.int32)
            lines = lines_of(t)
            want_p[cu[b] : cu[b + 1]] = torch.tensor([starts[b] + len(x) - 1 for x in lines])
            want_m[cu[b] : cu[b + 1]] = packed(lines, words)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    masks = torch.full((n, words), 5, dtype=torch.int64, device="cuda")
    positions = torch.full((n,), 5, dtype=torch.int64, device="cuda")
    got = ops.tree_layout(parents.cuda(), torch.tensor(cu, dtype=torch.int32).cuda(),
                          torch.tensor(starts, dtype=torch.int32).cuda(), max_new, err, positions, masks)  # fmt: skip
    assert got[0] is positions and got[1] is masks
    assert torch.equal(positions.cpu(), want_p)
    assert torch.equal(masks.cpu(), want_m)
    assert int(err) == 0


@pytest.mark.parametrize("nodes", [1, 2, 3, 63, 64, 65, 127, 128, 129, 200, 257, 1000])
@pytest.mark.parametrize("line", [False, True])
def test_sizes(nodes, line):
    check([grown(nodes, nodes, line=line)], [nodes * 7])


def test_batches():
    trees = [grown(n, n, roots=min(n, 1 + n % 3)) for n in (5, 0, 70, 1, 64, 0, 33, 129)]
    check(trees, list(range(0, 800, 100)), before=3, behind=5)
    check(trees, list(range(0, 800, 100)), before=200, behind=100, max_new=300, words=6)
    check([grown(1 + i % 90, i) for i in range(500)], list(range(500)))


def test_every_node_a_root():
    check([[-1] * 130, [-1] * 3], [10, 0])


def test_empty_calls():
    positions, masks = ops.tree_layout(*(torch.zeros(n, dtype=torch.int32, device="cuda") for n in (0, 1, 0)), 4)
    assert positions.shape == (0,) and masks.shape == (0, 1)
    positions, masks = ops.tree_layout(torch.zeros(7, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"),
                                       torch.zeros(0, dtype=torch.int32, device="cuda"), 4)  # fmt: skip
    assert positions.tolist() == [0] * 7 and masks.flatten().tolist() == [0] * 7


@pytest.mark.parametrize("bad,node", [(-2, 1), (3, 3), (4, 2), (2**31 - 1, 0), (70, 66)])
def test_bad_parents_count_as_none(bad, node):
    tree = grown(80, 1)
    want = list(tree)
    tree[node], want[node] = bad, -1
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    positions, masks = ops.tree_layout(i32(tree), i32([0, 80]), i32([9]), 80, err)
    assert int(err) == _lib.DEVERR_PARENT
    assert torch.equal(masks.cpu(), packed(lines_of(want), 2))
    assert positions.tolist() == [9 + len(x) - 1 for x in lines_of(want)]


def test_sequences_that_do_not_fit_are_flagged_and_left_alone():
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for cu, start, max_new in (([0, 5, 12], [1, 2], 6), ([0, 5, 13], [1, 2], 9), ([0, 5, 12], [1, -2], 9)):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        positions = torch.full((12,), 5, dtype=torch.int64, device="cuda")
        got, masks = ops.tree_layout(i32([-1, 0, 0, 1, 1, -1, 0, 1, 2, 3, 4, 5]), i32(cu), i32(start), max_new, err, positions)
        assert int(err) == _lib.DEVERR_LENGTH
        assert got.tolist() == [1, 2, 2, 3, 3] + [5] * 7
        assert masks[:5, 0].tolist() == [1, 3, 5, 11, 19]


def test_graph_and_streams():
    trees = [grown(n, n) for n in (40, 70, 3)]
    cu = torch.tensor([0, 40, 110, 113], dtype=torch.int32).cuda()
    starts = torch.tensor([3, 4, 5], dtype=torch.int32).cuda()
    parents = torch.tensor(sum(trees, []), dtype=torch.int32).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.tree_layout(parents, cu, starts, 70)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        positions, masks = ops.tree_layout(parents, cu, starts, 70)
    for turn in range(3):
        trees = [grown(n, n + 50 * turn) for n in (40, 70, 3)]
        parents.copy_(torch.tensor(sum(trees, []), dtype=torch.int32))
        graph.replay()
        want = ops.tree_layout(parents, cu, starts, 70)
        torch.cuda.synchronize()
        assert torch.equal(positions, want[0]) and torch.equal(masks, want[1])
        assert torch.equal(masks.cpu(), torch.cat([packed(lines_of(t), 2) for t in trees]))
