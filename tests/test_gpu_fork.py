"""Forked and compacted caches go on as untouched ones do: the same logits, bit for bit."""

from __future__ import annotations

import random

import pytest
import torch

from tokquay_amd import kv_cache
from tokquay_amd.generate import paged_forward
from tokquay_amd.kv_cache import BlockAllocator
from tokquay_amd.model import GPT2, GPT2Config
from tokquay_amd.sequence import Sequence
from tokquay_amd.weights import random_state_dict

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    cfg = GPT2Config(n_layer=2)
    m = GPT2(cfg)
    m.load_state_dict(random_state_dict(cfg, seed=0))
    return m.cuda().eval()


@pytest.mark.parametrize("cut", [None, 33, 32, 5])
def test_a_fork_goes_on_as_a_sequence_of_its_own(model, cut):
    rng = random.Random(1)
    prompt = [rng.randrange(50256) for _ in range(45)]
    alloc = BlockAllocator(model.cfg, 64, 16, device="cuda")
    alloc.pool.fill_(float("nan"))  # nothing but what was written or copied is read
    parent = Sequence(0, list(prompt))
    alloc.allocate(parent)
    paged_forward(model, alloc, [parent])
    n = 45 if cut is None else cut
    child, plain = Sequence(1, prompt[:n] + [7, 11]), Sequence(2, prompt[:n] + [7, 11])
    alloc.fork(parent, child, cut)
    alloc.append_slot(child)
    # The child's tokens on the forked cache; a sequence of its own whose cache was computed the same way (the prompt at once).
    whole = Sequence(3, list(prompt))
    alloc.allocate(whole)
    paged_forward(model, alloc, [whole])
    alloc.allocate(plain)
    for i in range(n):
        a, b = whole.block_table[i // 16], plain.block_table[i // 16]
        alloc.pool[b, :, :, :, i % 16] = alloc.pool[a, :, :, :, i % 16]
    plain.num_cached_tokens = n
    got, want = paged_forward(model, alloc, [child]), paged_forward(model, alloc, [plain])
    assert torch.isfinite(got).all() and torch.equal(got, want)
    # The parent has not noticed, and goes on too.
    for s in (parent, whole):
        s.append_token(99)
        alloc.append_slot(s)
    got, want = paged_forward(model, alloc, [parent]), paged_forward(model, alloc, [whole])
    assert torch.isfinite(got).all() and torch.equal(got, want)
    alloc.check_device_errors()


def test_a_compacted_cache_goes_on(model):
    rng = random.Random(2)
    alloc = BlockAllocator(model.cfg, 64, 16, device="cuda")
    seqs = [Sequence(i, [rng.randrange(50256) for _ in range(rng.randint(10, 90))]) for i in range(8)]
    for s in seqs:
        alloc.allocate(s)
        paged_forward(model, alloc, [s])
    child = Sequence(8, seqs[5].token_ids + [3])
    alloc.fork(seqs[5], child)
    alloc.append_slot(child)
    for i in (0, 1, 4):
        alloc.free(seqs[i])
    live = [s for s in seqs if s.block_table]
    for s in live:
        s.append_token(5)
        alloc.append_slot(s)
    live.append(child)
    pool, tables, starts = alloc.pool.clone(), [list(s.block_table) for s in live], [s.num_cached_tokens for s in live]
    want = paged_forward(model, alloc, live)
    # The same step again, after the blocks have moved.
    alloc.pool.copy_(pool)
    for s, n in zip(live, starts):
        s.num_cached_tokens = n
    assert alloc.compact(live) > 0 and [s.block_table for s in live] != tables
    alloc.pool[alloc.num_used_blocks :] = float("nan")
    got = paged_forward(model, alloc, live)
    assert torch.isfinite(got).all() and torch.equal(got, want)
    alloc.check_device_errors()


def test_many_blocks_are_moved_by_several_calls(monkeypatch):
    monkeypatch.setattr(kv_cache, "COPY_PAIRS", 3)
    alloc = BlockAllocator(GPT2Config(n_layer=1, n_embd=64, n_head=1), 24, 4, device="cuda")
    alloc.pool.copy_(torch.randn(alloc.pool.shape, generator=torch.Generator().manual_seed(3)))
    first, second = Sequence(0, [0] * 48), Sequence(1, [0] * 41)
    for s in (first, second):
        alloc.allocate(s)
        s.num_cached_tokens = len(s.token_ids)
    want = alloc.pool[second.block_table].clone()
    alloc.free(first)
    assert alloc.compact([second]) == 11 and sorted(second.block_table) == list(range(11))
    assert torch.equal(alloc.pool[second.block_table], want)
    alloc.check_device_errors()


def test_a_fork_that_the_copy_refuses_changes_nothing():
    # Heads of 32: blocks of such a pool are shared, but not copied.
    alloc = BlockAllocator(GPT2Config(n_layer=1, n_embd=32, n_head=1), 8, 4, device="cuda")
    seq, child = Sequence(0, [0] * 10), Sequence(1, [0] * 10)
    alloc.allocate(seq)
    seq.num_cached_tokens = 10
    before = list(alloc.ref_counts), list(alloc._free)
    with pytest.raises(ValueError, match="copy_blocks"):
        alloc.fork(seq, child)
    assert child.block_table == [] and child.num_cached_tokens == 0 and (alloc.ref_counts, alloc._free) == before
    alloc.fork(seq, child, 8)
    assert child.block_table == seq.block_table[:2] and child.num_cached_tokens == 8
