"""accept_tree against a walk on the host: whole numbers and copied rows, equal."""

from __future__ import annotations

import random

import pytest
import torch

from tests.tree_cases import accepted, grown, moved
from tokquay_amd import _lib, ops

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, sizes, starts, layers=2, kv_heads=2, dim=64, dtype=torch.bfloat16, bs=16, seed=0, agree=0.85, line=False,
                 before=0, behind=0):  # fmt: skip
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        parents, drafts, tokens = [-1] * before, [0] * before, [0] * before
        self.cu = [before]
        for n in sizes:
            tree = grown(n, rng.randrange(10**9), line=line)
            mine = [rng.randrange(40) for _ in tree]  # few: siblings may be the same token
            children = [[i for i, p in enumerate(tree) if p == a] for a in range(n)]
            tokens += [mine[rng.choice(c)] if c and rng.random() < agree else rng.randrange(1000) for c in children]
            parents += tree
            drafts += mine
            self.cu.append(self.cu[-1] + n)
        parents, drafts, tokens = parents + [0] * behind, drafts + [0] * behind, tokens + [0] * behind
        self.parents = torch.tensor(parents, dtype=torch.int32)
        self.drafts, self.tokens = torch.tensor(drafts, dtype=torch.int64), torch.tensor(tokens, dtype=torch.int64)
        self.start = torch.tensor(starts, dtype=torch.int32)
        need = [-(-(s + n) // bs) for s, n in zip(starts, sizes)]
        ids = torch.randperm(sum(need) + 3, generator=g).int()
        self.tables = torch.zeros(len(sizes), max([1] + need) + 1, dtype=torch.int32)
        at = 0
        for b, k in enumerate(need):
            self.tables[b, :k] = ids[at : at + k]
            at += k
        self.pool = torch.randn(sum(need) + 3, layers, 2, kv_heads, bs, dim, generator=g).to(dtype)
        self.width = max([1] + list(sizes))

    def run(self, max_path=None, pool=True, err=None):
        max_path = max_path or self.width
        pool = self.pool.cuda() if pool else None
        more = {} if pool is None else {"pool": pool, "block_tables": self.tables.cuda(), "q_start": self.start.cuda()}
        got = ops.accept_tree(self.tokens.cuda(), self.drafts.cuda(), self.parents.cuda(),
                              torch.tensor(self.cu, dtype=torch.int32).cuda(), max_path, d_error=err, **more)  # fmt: skip
        return [t.cpu() for t in got] + [None if pool is None else pool.cpu()]

    def check(self, max_path=None, pool=True):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = self.run(max_path, pool, err)
        want = accepted(self.tokens, self.drafts, self.parents, self.cu, max_path or self.width)
        for g, w in zip(got, want):
            assert torch.equal(g, w)
        if pool:
            assert torch.equal(got[3], moved(self.pool, self.tables, self.start, want[1], want[2]))
        assert int(err) == 0
        return want


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("layers,kv_heads", [(1, 1), (3, 2), (12, 12)])
def test_pools(layers, kv_heads, dim, dtype):
    Case([26, 1, 9, 0, 40], [700, 3, 0, 5, 33], layers, kv_heads, dim, dtype, seed=1).check()


@pytest.mark.parametrize("bs", [1, 3, 8, 16, 64, 1024])
def test_block_sizes(bs):
    Case([30, 12, 64], [70, 0, 31], bs=bs, seed=2).check()


@pytest.mark.parametrize("nodes", [1, 2, 63, 64, 65, 130, 300])
def test_sizes(nodes):
    for seed in range(4):
        Case([nodes], [11], seed=seed).check()


def test_long_paths():
    # Lines that stand to the end: nothing moves; with a detour in front everything does.
    for nodes in (64, 65, 200):
        want = Case([nodes], [5], seed=3, agree=1.0, line=True).check()
        assert int(want[2]) == nodes
        c = Case([nodes + 1], [5], seed=4, agree=1.0, line=True)
        c.parents = torch.tensor([-1, 0] + [0] + list(range(2, nodes)), dtype=torch.int32)
        c.drafts = torch.arange(100, 101 + nodes)
        c.tokens = torch.cat([torch.tensor([102, 0]), torch.arange(103, 102 + nodes)])
        want = c.check()
        assert int(want[2]) == nodes and want[1][0, 1] == 2


def test_max_path():
    for max_path in (1, 2, 3, 100):
        Case([40, 80, 64], [5, 60, 700], seed=5, agree=1.0).check(max_path)
        Case([40, 80, 64], [5, 60, 700], seed=5, agree=1.0, line=True).check(max_path)


def test_without_a_pool():
    Case([26, 1, 9, 0, 40], [0] * 5, seed=6, before=4, behind=6).check(pool=False)


def test_batches_and_rows_around():
    rng = random.Random(7)
    sizes = [rng.randrange(0, 70) for _ in range(200)]
    Case(sizes, [rng.randrange(0, 60) for _ in sizes], seed=7, before=3, behind=9).check()


def test_first_of_equal_children_and_no_negative_tokens():
    c = Case([5], [0], seed=8)
    c.parents = torch.tensor([-1, 0, 0, 1, 2], dtype=torch.int32)
    c.drafts = torch.tensor([9, 4, 4, 6, 7])
    c.tokens = torch.tensor([4, 6, 7, -1, 3])
    assert c.check()[1].tolist() == [[0, 1, 3, -1, -1]]
    c.drafts = torch.tensor([9, -1, 4, 6, 7])
    c.tokens = torch.tensor([-1, 6, 7, 1, 3])
    assert c.check()[1].tolist() == [[0, -1, -1, -1, -1]]


def test_nodes_before_their_parents_are_not_looked_at():
    c = Case([4], [0], seed=9)
    c.parents = torch.tensor([-1, 2, 0, 2], dtype=torch.int32)  # node 1 before its parent
    c.drafts = torch.tensor([9, 5, 4, 5])
    c.tokens = torch.tensor([4, 5, 5, 8])
    assert c.check()[1].tolist() == [[0, 2, 3, -1]]
    c.parents = torch.tensor([0, 1, 2, 3], dtype=torch.int32)  # each its own
    c.drafts = c.tokens = torch.tensor([4, 4, 4, 4])
    assert c.check()[1].tolist() == [[0, -1, -1, -1]]


def test_errors_are_flagged():
    c = Case([20, 30], [5, 9], seed=10)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = c.run()
    c.cu[2] = 60  # past the rows
    tokens, path, counts, pool = c.run(err=err)
    assert int(err) == _lib.DEVERR_LENGTH
    assert int(counts[1]) == 0 and bool((tokens[1] == -1).all()) and bool((path[1] == -1).all())
    assert torch.equal(tokens[0], want[0][0])
    c.cu[2] = 50
    for start in (-1, 16 * c.tables.size(1) - 29):
        err.zero_()
        c.start[1] = start
        tokens, path, counts, pool = c.run(err=err)
        assert int(err) == _lib.DEVERR_LENGTH and int(counts[1]) == 0
    # A bad block: the rows that need it stay where they are, the others move.
    c = Case([64], [0], seed=11, agree=1.0)
    want = accepted(c.tokens, c.drafts, c.parents, c.cu, 64)
    n = int(want[2][0])
    assert not torch.equal(want[1][0, :n], torch.arange(n, dtype=torch.int32))  # something would move
    c.tables[0] = c.pool.size(0)
    err.zero_()
    tokens, path, counts, pool = c.run(err=err)
    assert int(err) == _lib.DEVERR_BLOCK_ID
    assert torch.equal(path, want[1]) and torch.equal(pool, c.pool)


def test_positions_end_before_2_31():
    # A block table of more positions than 32 bits count, all in one block: the last sequence that fits them, and those that do not.
    bs, blocks = 1024, (1 << 21) + 1
    c = Case([8], [0], layers=1, kv_heads=1, bs=bs, seed=14)
    c.parents = torch.tensor([-1, 0, 0, 1, 2, 2, 3, 5], dtype=torch.int32)
    c.drafts = torch.tensor([1, 2, 3, 4, 5, 6, 7, 8])
    c.tokens = torch.tensor([3, 0, 6, 0, 0, 8, 0, 0])
    c.tables = torch.zeros(1, blocks, dtype=torch.int32)
    for start in (2**31 - 1 - 8, 2**31 - 8, 2**31 - 6, 2**31 - 1):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        c.start[0] = start
        tokens, path, counts, pool = c.run(err=err)
        if start + 8 < 2**31:
            assert path.tolist() == [[0, 2, 5, 7, -1, -1, -1, -1]] and tokens.tolist() == [[3, 6, 8, 0, -1, -1, -1, -1]]
            want = c.pool.clone()
            for j, node in enumerate([0, 2, 5, 7]):
                want[0, :, :, :, (start + j) % bs] = c.pool[0, :, :, :, (start + node) % bs]
            assert torch.equal(pool, want) and int(err) == 0
        else:
            assert int(err) == _lib.DEVERR_LENGTH and counts.tolist() == [0] and bool((path == -1).all())
            assert bool((tokens == -1).all()) and torch.equal(pool, c.pool)


def test_large_pools():
    # Blocks past 2^31 bytes and elements.
    c = Case([30, 40], [40, 3], layers=2, kv_heads=8, dim=128, seed=12, agree=1.0)
    block = c.pool[0].numel()
    blocks = 2**32 // block + 50
    shift = blocks - c.pool.size(0)
    pool = torch.zeros(blocks, *c.pool.shape[1:], dtype=c.pool.dtype, device="cuda")
    pool[shift:] = c.pool.cuda()
    want = accepted(c.tokens, c.drafts, c.parents, c.cu, 40)
    ops.accept_tree(c.tokens.cuda(), c.drafts.cuda(), c.parents.cuda(), torch.tensor(c.cu, dtype=torch.int32).cuda(), 40, pool,
                    (c.tables + shift).cuda(), c.start.cuda())  # fmt: skip
    assert torch.equal(pool[shift:].cpu(), moved(c.pool, c.tables, c.start, want[1], want[2]))


def test_graphs():
    c = Case([26, 40, 9], [70, 3, 20], seed=13)
    tokens, drafts, parents = c.tokens.cuda(), c.drafts.cuda(), c.parents.cuda()
    cu, pool, tables, start = torch.tensor(c.cu, dtype=torch.int32).cuda(), c.pool.cuda(), c.tables.cuda(), c.start.cuda()
    ops.accept_tree(tokens, drafts, parents, cu, 40, pool, tables, start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.accept_tree(tokens, drafts, parents, cu, 40, pool, tables, start)
    for turn in range(3):
        other = Case([26, 40, 9], [70, 3, 20], seed=20 + turn)
        for a, b in ((tokens, other.tokens), (drafts, other.drafts), (parents, other.parents), (pool, c.pool)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = accepted(other.tokens, other.drafts, other.parents, c.cu, 40)
        for g, w in zip(got, want):
            assert torch.equal(g.cpu(), w)
        assert torch.equal(pool.cpu(), moved(c.pool, c.tables, c.start, want[1], want[2]))
