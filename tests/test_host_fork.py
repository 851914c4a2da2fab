"""BlockAllocator.fork and compact on the CPU: tables, ref counts, free list and the pool's contents."""

from __future__ import annotations

import random

import pytest
import torch

from tokquay_amd.kv_cache import BlockAllocator, OutOfBlocksError
from tokquay_amd.model import GPT2Config
from tokquay_amd.scheduler import RequestRejected, Scheduler, SchedulerConfig
from tokquay_amd.sequence import Sequence

TINY = GPT2Config(vocab_size=8, n_positions=64, n_embd=4, n_layer=2, n_head=1)


def allocator(num_blocks=12, block_size=4):
    a = BlockAllocator(TINY, num_blocks, block_size, device="cpu")
    a.pool.copy_(torch.randn(a.pool.shape, generator=torch.Generator().manual_seed(0)))
    return a


def sequence(a, i, tokens):
    s = Sequence(i, [0] * tokens)
    a.allocate(s)
    s.num_cached_tokens = tokens
    return s


def cached(a, s):
    """What the cache holds of a sequence, [positions, layers, 2, heads, d]."""
    rows = [a.pool[s.block_table[i // a.block_size], :, :, :, i % a.block_size] for i in range(s.num_cached_tokens)]
    return torch.stack(rows) if rows else a.pool.new_zeros(0, *a.pool.shape[1:4], a.pool.size(5))


@pytest.mark.parametrize("n", [0, 1, 3, 4, 5, 8, 10, None])
def test_fork(n):
    a = allocator()
    s, child = sequence(a, 0, 10), Sequence(1, [0] * 10)
    before = cached(a, s)
    a.fork(s, child, n)
    n = 10 if n is None else n
    assert child.num_cached_tokens == n and len(child.block_table) == a.blocks_needed(n)
    assert torch.equal(cached(a, child), before[:n]) and torch.equal(cached(a, s), before)
    assert child.block_table[: n // 4] == s.block_table[: n // 4]
    assert not set(child.block_table[n // 4 :]) & set(s.block_table)
    assert a.num_used_blocks == 3 + (n % 4 > 0)
    # Either may end first, and each goes on in blocks of its own.
    a.append_slot(child, n + 1)
    assert child.block_table[n // 4] not in s.block_table
    a.free(s)
    assert torch.equal(cached(a, child), before[:n])
    a.free(child)
    assert a.num_free_blocks == 12 and not any(a.ref_counts)


def test_forks_of_forks_share_until_the_last_is_freed():
    a = allocator()
    s = sequence(a, 0, 9)
    children = [Sequence(i, [0] * 9) for i in range(1, 4)]
    a.fork(s, children[0])
    a.fork(children[0], children[1], 8)
    a.fork(s, children[2], 4)
    assert [a.ref_counts[b] for b in s.block_table] == [4, 3, 1]
    for q in [children[1], s, children[0]]:
        a.free(q)
    assert [a.ref_counts[b] for b in children[2].block_table] == [1] and a.num_used_blocks == 1


def test_refused_forks_change_nothing():
    a = allocator(num_blocks=3)
    s, child = sequence(a, 0, 10), Sequence(1, [0])
    before = a.pool.clone(), list(a.ref_counts), a.num_free_blocks
    with pytest.raises(OutOfBlocksError):
        a.fork(s, child)
    for n in (-1, 11):
        with pytest.raises(ValueError, match="cached tokens"):
            a.fork(s, child, n)
    with pytest.raises(ValueError, match="already owns blocks"):
        a.fork(child, s, 0)
    assert child.block_table == [] and child.num_cached_tokens == 0
    assert torch.equal(a.pool, before[0]) and a.ref_counts == before[1] and a.num_free_blocks == before[2]


def test_compact():
    rng = random.Random(0)
    a = allocator(num_blocks=40)
    seqs = [sequence(a, i, rng.randint(1, 14)) for i in range(9)]
    child = Sequence(9, [0] * 14)
    a.fork(seqs[4], child)
    for i in (0, 2, 3, 7):
        a.free(seqs[i])
    seqs = [s for s in seqs if s.block_table] + [child]
    before = [cached(a, s) for s in seqs]
    counts = sorted(c for c in a.ref_counts if c)
    used = a.num_used_blocks
    with pytest.raises(ValueError, match="in use"):
        a.compact(seqs[1:-1])
    assert a.compact(seqs) > 0
    assert {b for s in seqs for b in s.block_table} == set(range(used))
    assert all(torch.equal(cached(a, s), x) for s, x in zip(seqs, before))
    assert sorted(c for c in a.ref_counts if c) == counts and a.num_used_blocks == used
    assert a.compact(seqs) == 0
    more = sequence(a, 20, 4)
    assert more.block_table == [used]
    for s in seqs + [more]:
        a.free(s)
    assert a.num_free_blocks == 40 and a.compact([]) == 0


def shared(cuts):
    """An allocator, a sequence behind freed blocks, and forks of it at the given cuts."""
    a = allocator(num_blocks=16)
    first, s = sequence(a, 0, 8), sequence(a, 1, 8)
    children = []
    for i, n in enumerate(cuts):
        children.append(Sequence(2 + i, [0] * 8))
        a.fork(s, children[-1], n)
    a.free(first)
    return a, s, children


@pytest.mark.parametrize("cuts", [[8], [4], [8, 8], [8, 4, 8]])
def test_compact_refuses_owners_left_out(cuts):
    # All blocks of a fork that was cut between two blocks belong to its parent too: without it no block is missing.
    a, s, children = shared(cuts)
    everyone = [s, *children]
    before = a.pool.clone(), [list(q.block_table) for q in everyone], list(a.ref_counts), list(a._free)
    for left_out in range(len(everyone)):
        given = everyone[:left_out] + everyone[left_out + 1 :]
        with pytest.raises(ValueError, match="in use"):
            a.compact(given)
        with pytest.raises(ValueError, match="in use"):  # one that is named twice does not stand for the other
            a.compact(given + given[:1])
    assert torch.equal(a.pool, before[0]) and [q.block_table for q in everyone] == before[1]
    assert a.ref_counts == before[2] and a._free == before[3]
    contents = [cached(a, q) for q in everyone]
    assert a.compact(everyone + [s]) == 2
    assert all(torch.equal(cached(a, q), x) for q, x in zip(everyone, contents))
    for q in everyone:
        a.free(q)
    assert a.num_free_blocks == 16 and not any(a.ref_counts)


def test_compact_refuses_blocks_that_are_free():
    a, s, _ = shared([])
    stale = Sequence(9, [0])
    stale.block_table = [15]
    with pytest.raises(ValueError, match="in use"):
        a.compact([s, stale])


def test_a_fork_whose_copy_is_refused_changes_nothing(monkeypatch):
    a = allocator()
    s, child = sequence(a, 0, 10), Sequence(1, [0] * 10)
    before = list(a.ref_counts), list(a._free), list(s.block_table)

    def refuse(*args):
        raise ValueError("copy_blocks: pool has another head size")

    monkeypatch.setattr(a, "_copy", refuse)
    with pytest.raises(ValueError, match="another head size"):
        a.fork(s, child)
    assert child.block_table == [] and child.num_cached_tokens == 0
    assert (list(a.ref_counts), list(a._free), list(s.block_table)) == before


def test_the_scheduler_refuses_sequences_that_own_blocks():
    # A queued sequence has none: it gets blocks for all of its tokens when it is admitted.
    a = allocator()
    s, child = sequence(a, 0, 9), Sequence(1, [0] * 10)
    sched = Scheduler(a, SchedulerConfig(max_model_len=64, max_num_batched_tokens=64, watermark_blocks=0))
    a.fork(s, child)
    with pytest.raises(RequestRejected, match="already owns blocks"):
        sched.add_request(child)
    assert not sched.has_unfinished() and a.num_used_blocks == 4
    a.free(child)
    child.num_cached_tokens = 0
    sched.add_request(child)
    a.fork(s, child, 8)  # behind the queue's back: it says so, and loses nothing
    with pytest.raises(ValueError, match="already owns blocks"):
        sched.schedule()
    assert len(sched.waiting) == 1 and sched.waiting[0] is child and not sched.running
    sched.abort(child)
    assert a.num_used_blocks == 3 and not sched.has_unfinished()


def test_the_scheduler_refuses_cached_tokens_without_blocks():
    # A fork that gave its blocks back still counts its cached tokens: admitted, it would read them from blocks that nobody has written.
    a = allocator()
    s, child = sequence(a, 0, 9), Sequence(1, [0] * 10)
    sched = Scheduler(a, SchedulerConfig(max_model_len=64, max_num_batched_tokens=64, watermark_blocks=0))
    a.fork(s, child)
    a.free(child)
    with pytest.raises(RequestRejected, match="cached tokens"):
        sched.add_request(child)
    child.reset_for_recompute()
    sched.add_request(child)
    assert sched.schedule().seqs == [child]
