"""copy_blocks against indexing on the host: equal."""

from __future__ import annotations

import pytest
import torch

from tokquay_amd import _lib, ops

pytestmark = pytest.mark.gpu


def make(blocks, layers=2, kv_heads=2, bs=16, dim=64, dtype=torch.bfloat16, seed=0):
    return torch.randn(blocks, layers, 2, kv_heads, bs, dim, generator=torch.Generator().manual_seed(seed)).to(dtype)


def copied(pool, src, dst, slots=None):
    new = pool.clone()
    for i, (s, d) in enumerate(zip(src, dst)):
        n = pool.size(4) if slots is None else slots[i]
        new[d, ..., :n, :] = pool[s, ..., :n, :]
    return new


def run(pool, src, dst, slots=None, err=None):
    got = pool.cuda()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.copy_blocks(got, i32(src), i32(dst), None if slots is None else i32(slots), err)
    return got.cpu()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layers,kv_heads,bs,dim", [(1, 1, 1, 64), (2, 3, 16, 128), (12, 12, 16, 64), (3, 1, 7, 64), (2, 2, 1024, 128)])
def test_pools(layers, kv_heads, bs, dim, dtype):
    pool = make(9, layers, kv_heads, bs, dim, dtype)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    src, dst = [4, 0, 7], [2, 8, 5]
    assert torch.equal(run(pool, src, dst, None, err), copied(pool, src, dst))
    slots = [bs, max(1, bs // 2), 1]
    assert torch.equal(run(pool, src, dst, slots, err), copied(pool, src, dst, slots))
    assert int(err) == 0


def test_one_source_to_many():
    pool = make(20)
    src, dst = [3] * 12, [i for i in range(4, 16)]
    slots = list(range(1, 13))
    assert torch.equal(run(pool, src, dst, slots), copied(pool, src, dst, slots))


@pytest.mark.parametrize("pairs", [1, 255, 256, 257, 1000])
def test_many_pairs(pairs):
    pool = make(2 * pairs + 5, 1, 1, 4)
    ids = torch.randperm(2 * pairs + 5, generator=torch.Generator().manual_seed(pairs)).tolist()
    src, dst = ids[:pairs], ids[pairs : 2 * pairs]
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert torch.equal(run(pool, src, dst, None, err), copied(pool, src, dst))
    assert int(err) == 0


def test_pairs_that_do_nothing():
    pool = make(8)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    # Padding, a block to itself, no slots: also where other pairs write or read those blocks.
    got = run(pool, [-1, 2, -1, 3, 5, 6], [4, -1, -1, 3, 4, 3], [16, 16, 16, 16, 0, 16], err)
    assert torch.equal(got, copied(pool, [6], [3]))
    assert int(err) == 0
    assert torch.equal(run(pool, [], []), pool)


def test_copies_that_meet_are_flagged_and_left_out():
    pool = make(12)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    # 1 -> 2 would write what 2 -> 3 reads; of 4 -> 5 and 6 -> 5 the first is made; 7 -> 8 and 8 -> 7 both meet.
    got = run(pool, [1, 2, 4, 6, 7, 8, 9], [2, 3, 5, 5, 8, 7, 10], None, err)
    assert int(err) == _lib.DEVERR_OVERLAP
    assert torch.equal(got, copied(pool, [2, 4, 9], [3, 5, 10]))
    err.zero_()
    pool = make(700, 1, 1, 4)
    src, dst = list(range(300)) + [650, 5], list(range(300, 600)) + [300, 650]
    got = run(pool, src, dst, None, err)
    assert int(err) == _lib.DEVERR_OVERLAP
    assert torch.equal(got, copied(pool, src[:300], dst[:300]))


def test_bad_ids_and_counts_are_flagged():
    pool = make(6)
    for src, dst, slots, bits in (([6, 0], [1, 2], [1, 1], _lib.DEVERR_BLOCK_ID), ([1, 0], [2**31 - 1, 2], [1, 1], _lib.DEVERR_BLOCK_ID),
                                  ([1, 0], [3, 2], [17, 1], _lib.DEVERR_LENGTH), ([1, 0], [3, 2], [-1, 1], _lib.DEVERR_LENGTH)):  # fmt: skip
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        assert torch.equal(run(pool, src, dst, slots, err), copied(pool, [0], [2], [1]))
        assert int(err) == bits


def test_large_pools():
    # Blocks past 2^32 bytes.
    pool = torch.zeros(2**33 // 2**21 + 6, 16, 2, 8, 16, 128, dtype=torch.float32, device="cuda")
    n = pool.size(0)
    pool[n - 1] = torch.randn(pool.shape[1:], device="cuda")
    pool[2] = torch.randn(pool.shape[1:], device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.copy_blocks(pool, i32([n - 1, 2]), i32([1, n - 3]))
    assert torch.equal(pool[1], pool[n - 1]) and torch.equal(pool[n - 3], pool[2])
    assert int(torch.count_nonzero(pool[n - 2])) == 0 and int(torch.count_nonzero(pool[0])) == 0


def test_graphs():
    pool = make(10).cuda()
    old = pool.clone()
    src, dst, slots = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([1, 2, 3], [4, 5, 6], [16, 3, 9]))
    ops.copy_blocks(pool, src, dst, slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_blocks(pool, src, dst, slots)
    for turn in range(3):
        pool.copy_(old)
        src.copy_(torch.tensor([turn, 2, -1]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool.cpu(), copied(old.cpu(), [turn, 2], [4, 5], [16, 3]))
