"""verify_drafts against the accept / resample rule in float64 on the host: whole numbers, equal."""

from __future__ import annotations

import math

import pytest
import torch

from tests.chunk_cases import verified
from tokquay_amd import _lib, ops

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, drafts, vocab, dtype=torch.float32, probs=True, temps=(1.0,), seed=0, spread=3.0, near=0.5):
        g = torch.Generator().manual_seed(seed)
        cu = [0]
        for n in drafts:
            cu.append(cu[-1] + n)
        rows = cu[-1]
        self.cu = torch.tensor(cu, dtype=torch.int32)
        self.temperature = torch.tensor([temps[b % len(temps)] for b in range(len(drafts))])
        self.logits = (torch.randn(rows, vocab, generator=g) * spread).to(dtype)
        other = self.logits.float() + torch.randn(rows, vocab, generator=g) * near
        owner = torch.repeat_interleave(torch.arange(len(drafts)), torch.tensor(drafts))
        t = self.temperature[owner][:, None]
        self.probs = None
        if probs:
            hard = torch.nn.functional.one_hot(other.argmax(-1), vocab).float()
            self.probs = torch.where(t > 0, torch.softmax(other / torch.where(t > 0, t, 1.0), -1), hard)
            self.drafts = torch.multinomial(self.probs, 1, generator=g)[:, 0] if rows else torch.zeros(0, dtype=torch.int64)
        else:
            self.drafts = other.argmax(-1)
        self.uniforms = torch.rand(rows, generator=g)
        self.max_rows = max([1] + list(drafts))

    def run(self, logits=None, probs=None, err=None, max_rows=None):
        p = self.probs if probs is None else probs
        tokens, accepted = ops.verify_drafts((self.logits if logits is None else logits).cuda(), self.drafts.cuda(),
                                             self.uniforms.cuda(), self.cu.cuda(), max_rows or self.max_rows,
                                             self.temperature.cuda(), None if p is None else p.cuda(), err)  # fmt: skip
        return tokens.cpu(), accepted.cpu()

    def check(self):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        tokens, accepted = self.run(err=err)
        want, count = verified(self.logits, self.drafts, self.uniforms, self.cu, self.max_rows, self.temperature, self.probs)
        assert torch.equal(accepted, count)
        assert torch.equal(tokens, want)
        return int(err)


# Rows of each sequence: its drafts and one more. 0: no rows.
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 255, 8192, 8193, 50257])
def test_vocabularies_and_types(vocab, probs, dtype):
    assert Case([5, 1, 3, 0, 8], vocab, dtype, probs, temps=(1.0, 0.7, 0.0), seed=vocab).check() == 0


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("seed", range(4))
def test_many_sequences(probs, seed):
    g = torch.Generator().manual_seed(seed)
    rows = torch.randint(0, 7, (150,), generator=g).tolist()
    assert Case(rows, 1013, torch.float32, probs, temps=(1.0, 0.6, 0.0, 1.3), seed=seed).check() == 0


@pytest.mark.parametrize("probs", [True, False])
def test_greedy_follows_the_argmax(probs):
    c = Case([6] * 20, 3001, torch.bfloat16, probs, temps=(0.0,), seed=3, near=0.0)
    c.check()
    tokens, accepted = c.run()
    assert bool((accepted == 5).all())
    assert torch.equal(tokens.flatten(), c.logits.float().argmax(-1))


def test_ties_go_to_the_lowest_column():
    c = Case([2, 2], 700, torch.bfloat16, False, temps=(0.0, 1.0), seed=4)
    c.logits[:] = 0.0
    c.drafts[:] = torch.tensor([0, 0, 699, 0])
    c.uniforms[:] = torch.tensor([0.5, 0.5, 0.9, 0.5])
    tokens, accepted = c.run()
    assert accepted.tolist() == [1, 0]
    # The second sequence: 699 equal weights are left (all but the draft's), and half their sum ends inside column 349.
    assert tokens.tolist() == [[0, 0], [349, -1]]


def test_many_rows_of_one_sequence():
    c = Case([300], 997, torch.float32, True, seed=5, near=0.02)
    c.uniforms[:299] *= 1e-6  # everything stands
    assert c.check() == 0
    assert int(c.run()[1]) == 299


def test_ends_of_the_unit_interval():
    for u in (0.0, 1 - 2.0**-24):
        c = Case([3, 1, 2], 5003, torch.float32, True, seed=6)
        c.uniforms[:] = u
        c.check()


def test_masked_tokens_are_never_drawn():
    c = Case([1] * 64, 9001, torch.float32, False, seed=7)
    c.logits[:, 3000:] = -math.inf
    c.logits[:, :17] = -math.inf
    c.check()
    tokens, _ = c.run()
    assert bool(((tokens >= 17) & (tokens < 3000)).all())


def test_one_token_left():
    c = Case([2] * 8, 20000, torch.float16, True, seed=8)
    c.logits[:] = -math.inf
    c.logits[:, 19999] = -5.0
    assert c.check() == 0
    assert bool((c.run()[0][:, 0] == 19999).all())


def test_nothing_left_of_the_difference():
    # q covers p everywhere (twice its values), and the draft does not stand: the draw is from p.
    c = Case([2] * 6, 12000, torch.float32, True, seed=9, near=0.0)
    c.probs = c.probs * 2
    c.uniforms[:] = torch.where(torch.arange(12) % 2 == 0, 0.9, c.uniforms)
    c.check()
    assert bool((c.run()[1] == 0).all())


def test_extreme_logits():
    c = Case([3] * 4, 9000, torch.float32, True, seed=10)
    c.logits *= 1e30
    c.check()
    c = Case([3] * 4, 9000, torch.float32, True, seed=10, temps=(1e-30, 1e30))
    c.check()


def test_rows_without_a_distribution_are_flagged_and_greedy():
    for spoil in (math.nan, math.inf):
        c = Case([3, 2, 2], 9000, torch.float32, True, seed=11)
        c.logits[1, 8500] = spoil
        c.uniforms[0] = 0.0  # the first draft stands: the row is come to
        assert c.check() == _lib.DEVERR_VALUE
    c = Case([2], 9000, torch.float32, True, seed=12)
    c.logits[1] = -math.inf
    c.uniforms[0] = 0.0
    assert c.check() == _lib.DEVERR_VALUE
    # Behind the first rejection nothing is come to; greedy sequences take NaN as the largest.
    c = Case([4], 500, torch.float32, False, seed=13)
    c.uniforms[0] = 1 - 2.0**-24
    c.logits[0] = 0.0
    c.logits[2, 5] = math.nan
    assert c.check() == 0
    c = Case([2], 500, torch.float32, False, temps=(0.0,), seed=14)
    c.logits[0, 77] = math.nan
    c.drafts[0] = 77
    assert c.check() == 0


def test_drafts_outside_the_vocabulary_do_not_stand():
    for x in (-1, 600, 2**40):
        for probs in (True, False):
            c = Case([3, 2], 600, torch.float32, probs, seed=15)
            c.drafts[0] = x
            assert c.check() == _lib.DEVERR_TOKEN


def test_sequences_that_do_not_fit_are_flagged():
    c = Case([3, 2, 4], 600, torch.float32, True, seed=16)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    tokens, accepted = c.run(err=err, max_rows=3)
    want, count = verified(c.logits, c.drafts, c.uniforms, c.cu, 4, c.temperature, c.probs)
    assert int(err) == _lib.DEVERR_LENGTH
    assert torch.equal(tokens[:2], want[:2, :3]) and torch.equal(accepted[:2], count[:2])
    assert tokens[2].tolist() == [-1, -1, -1] and int(accepted[2]) == 0
    c.cu[3] = 10  # past the rows
    err.zero_()
    c.run(err=err)
    assert int(err) == _lib.DEVERR_LENGTH


def test_no_sequences_and_no_rows():
    z = torch.zeros(0, device="cuda")
    tokens, accepted = ops.verify_drafts(torch.zeros(0, 50, device="cuda"), z.long(), z, torch.zeros(1, dtype=torch.int32, device="cuda"), 4, z)
    assert tokens.shape == (0, 4) and accepted.shape == (0,)
    c = Case([0, 0, 0], 600, seed=17)
    tokens, accepted = c.run()
    assert bool((tokens == -1).all()) and bool((accepted == 0).all())


def test_strided_rows():
    c = Case([3, 1, 4], 5001, torch.bfloat16, True, seed=18)
    logits = torch.zeros(8, 5100, dtype=torch.bfloat16, device="cuda")[:, 7 : 7 + 5001]
    probs = torch.zeros(8, 5050, device="cuda")[:, 3 : 3 + 5001]
    logits.copy_(c.logits)
    probs.copy_(c.probs)
    tokens, accepted = c.run(logits=logits, probs=probs)
    want, count = verified(c.logits, c.drafts, c.uniforms, c.cu, c.max_rows, c.temperature, c.probs)
    assert torch.equal(tokens, want) and torch.equal(accepted, count)


def test_drafts_and_draws_have_the_targets_distribution():
    # 40,000 independent steps of one draft over 6 tokens: the first token's counts against the target's (chi squared of 5
    # degrees: 30 is passed once in 10^5 tries).
    g = torch.Generator().manual_seed(19)
    n, vocab = 40000, 6
    target, draft = torch.randn(vocab, generator=g), torch.randn(vocab, generator=g)
    q = torch.softmax(draft, -1)
    drafts = torch.zeros(2 * n, dtype=torch.int64)
    drafts[::2] = torch.multinomial(q, n, replacement=True, generator=g)
    tokens, _ = ops.verify_drafts(target.repeat(2 * n, 1).cuda(), drafts.cuda(), torch.rand(2 * n, generator=g).cuda(),
                                  torch.arange(0, 2 * n + 1, 2, dtype=torch.int32).cuda(), 2, torch.ones(n).cuda(),
                                  q.repeat(2 * n, 1).cuda())  # fmt: skip
    p = torch.softmax(target.double(), -1)
    counts = torch.bincount(tokens[:, 0].cpu(), minlength=vocab).double()
    assert float(((counts - n * p) ** 2 / (n * p)).sum()) < 30


def test_two_streams_and_a_graph():
    a, b = Case([5, 3], 50257, torch.float32, True, seed=20), Case([5, 3], 50257, torch.float32, True, seed=21)
    put = [[t.cuda() for t in (c.logits, c.drafts, c.uniforms, c.cu, c.temperature, c.probs)] for c in (a, b)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for i, (l, d, u, cu, t, p) in enumerate(put):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.verify_drafts(l, d, u, cu, 5, t, p))
    torch.cuda.synchronize()
    wants = [verified(c.logits, c.drafts, c.uniforms, c.cu, 5, c.temperature, c.probs) for c in (a, b)]
    for i in range(2):
        for tokens, accepted in got[i]:
            assert torch.equal(tokens.cpu(), wants[i][0]) and torch.equal(accepted.cpu(), wants[i][1])
    l, d, u, cu, t, p = put[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, accepted = ops.verify_drafts(l, d, u, cu, 5, t, p)
    for i in (0, 1, 0, 1):
        c = (a, b)[i]
        for to, x in zip(put[0], (c.logits, c.drafts, c.uniforms, c.cu, c.temperature, c.probs)):
            to.copy_(x)
        tokens.zero_()
        graph.replay()
        assert torch.equal(tokens.cpu(), wants[i][0]) and torch.equal(accepted.cpu(), wants[i][1])


def test_refusals():
    c = Case([3, 2], 600, seed=22)
    good = dict(logits=c.logits.cuda(), draft_tokens=c.drafts.cuda(), uniforms=c.uniforms.cuda(), cu_seqlens_q=c.cu.cuda(),
                max_query_len=3, temperature=c.temperature.cuda(), draft_probs=c.probs.cuda())  # fmt: skip
    ops.verify_drafts(**good)
    for name, value in [("logits", c.logits.cuda().double()), ("logits", c.logits), ("draft_tokens", c.drafts.cuda().int()),
                        ("draft_tokens", c.drafts.cuda()[:-1]), ("uniforms", c.uniforms.cuda().double()),
                        ("cu_seqlens_q", c.cu.cuda().long()), ("temperature", c.temperature.cuda()[:1]), ("max_query_len", 0),
                        ("draft_probs", c.probs.cuda()[:, :-1]), ("draft_probs", c.probs.cuda().half()),
                        ("tokens", torch.zeros(2, 3, dtype=torch.int32, device="cuda")),
                        ("accepted", torch.zeros(3, dtype=torch.int32, device="cuda"))]:  # fmt: skip
        with pytest.raises(ValueError, match="verify_drafts"):
            ops.verify_drafts(**{**good, name: value})
    with pytest.raises(ValueError, match="tokens must be"):
        ops.verify_drafts(**good, tokens=torch.zeros(2, 4, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("sequences", [3, 200])
def test_a_draft_of_any_weight_is_left_out(sequences):
    # Drafts with between a thousandth of the weight and all but a millionth of it, none of which stands.
    c = Case([2] * sequences, 20000, torch.float32, False, seed=17)
    rows = torch.arange(0, 2 * sequences, 2)
    c.drafts[rows] = torch.arange(sequences) * 7919 % 20000
    c.logits[rows, c.drafts[rows]] = -math.inf
    others = torch.logsumexp(c.logits[rows], -1)
    c.logits[rows, c.drafts[rows]] = others + torch.linspace(-7.0, 14.0, sequences)
    c.uniforms[rows] = 1 - 2.0**-24
    assert c.check() == 0
    tokens, accepted = c.run()
    assert bool((accepted == 0).all())
    assert bool((tokens[:, 0] != c.drafts[rows]).all())


@pytest.mark.parametrize("probs", [True, False])
def test_thousands_of_sequences_each_by_its_temperature(probs):
    g = torch.Generator().manual_seed(23)
    rows = torch.randint(0, 3, (5000,), generator=g).tolist()
    assert Case(rows, 11, torch.float32, probs, temps=(0.5, 0.0, 1.0, 2.0, 0.25), seed=24).check() == 0


@pytest.mark.parametrize("probs", [True, False])
def test_a_captured_batch_replays(probs):
    # 130 sequences of 13 chunks of 4,096 columns: the decision is a launch of its own, with probabilities too.
    a, b = (Case([2] * 130, 50257, torch.bfloat16, probs, seed=s) for s in (25, 26))
    put = [None if t is None else t.cuda() for t in (a.logits, a.drafts, a.uniforms, a.cu, a.temperature, a.probs)]
    wants = [verified(c.logits, c.drafts, c.uniforms, c.cu, 2, c.temperature, c.probs) for c in (a, b)]
    l, d, u, cu, t, p = put
    ops.verify_drafts(l, d, u, cu, 2, t, p)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, accepted = ops.verify_drafts(l, d, u, cu, 2, t, p)
    for i in (0, 1, 0, 1):
        c = (a, b)[i]
        for to, x in zip(put, (c.logits, c.drafts, c.uniforms, c.cu, c.temperature, c.probs)):
            if to is not None:
                to.copy_(x)
        tokens.zero_()
        graph.replay()
        assert torch.equal(tokens.cpu(), wants[i][0]) and torch.equal(accepted.cpu(), wants[i][1])


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("cu", [[0, 99, 5, 9], [0, 5, -3, 9], [0, 5, 2, 7], [0, 3, 99, 9], [4, 0, 5, 9], [0, 2**31 - 1, 3, 9]])
@pytest.mark.parametrize("temps", [(1.0, 0.0, 0.8), (0.0, 1.0, 0.7), (0.9, 0.9, 0.9)])
def test_offsets_that_fall(cu, temps, probs):
    # A sequence beside one that does not fit gets its own result or is taken as one of no rows, never another's.
    c = Case([3, 2, 4], 600, torch.float32, probs, temps=temps, seed=16)
    c.cu = torch.tensor(cu, dtype=torch.int32)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    tokens, accepted = c.run(err=err, max_rows=5)
    assert int(err) == _lib.DEVERR_LENGTH
    for b in range(3):
        fits = 0 <= cu[b] < cu[b + 1] <= 9 and cu[b + 1] - cu[b] <= 5
        if fits and not (int(accepted[b]) == 0 and bool((tokens[b] == -1).all())):
            want, count = verified(c.logits, c.drafts, c.uniforms, c.cu[b : b + 2], 5, c.temperature[b : b + 1], c.probs)
            assert torch.equal(tokens[b], want[0]) and int(accepted[b]) == int(count[0])
        else:
            assert bool((tokens[b] == -1).all()) and int(accepted[b]) == 0


# draw of 16 columns a thread without a decision launch (the first four); of 32, without and with one; vocabularies whose
# statistics always take 32 columns a thread.
@pytest.mark.parametrize("sequences,vocab,dtype", [
    (64, 50257, torch.float32), (64, 50257, torch.bfloat16), (32, 128000, torch.float32), (17, 60001, torch.float16),
    (2, 1048577, torch.float32), (3, 2097152, torch.bfloat16), (13, 1100003, torch.float16), (2, 600011, torch.bfloat16),
])  # fmt: skip
@pytest.mark.parametrize("probs", [True, False])
def test_batches_and_vocabularies_of_every_draw(sequences, vocab, dtype, probs):
    rows = [(3 if vocab < 10**6 else 2) if b % 3 else 1 for b in range(sequences)]
    assert Case(rows, vocab, dtype, probs, temps=(1.0, 0.0, 0.8), seed=27).check() == 0
