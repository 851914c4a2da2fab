"""sample_tokens against ranking and drawing in float64 on the host: whole numbers, equal."""

from __future__ import annotations

import math

import pytest
import torch

from tests.tree_cases import sampled
from tokquay_amd import _lib, ops

pytestmark = pytest.mark.gpu

F32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


def settings(rows, users):
    """Columns of (temperature, top_k, top_p, min_p), row after row."""
    t, k, p, m = zip(*(users[r % len(users)] for r in range(rows)))
    return torch.tensor(t), torch.tensor(k, dtype=torch.int32), torch.tensor(p), torch.tensor(m)


def run(logits, uniforms, *rest, **more):
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    cuda = lambda t: t.cuda() if isinstance(t, torch.Tensor) else t  # noqa: E731
    got = ops.sample_tokens(cuda(logits), cuda(uniforms), *map(cuda, rest), d_error=err, **{k: cuda(v) for k, v in more.items()})
    return got.cpu(), int(err)


def check(logits, users, seed=0, uniforms=None):
    rows = logits.size(0)
    u = torch.rand(rows, generator=torch.Generator().manual_seed(seed)) if uniforms is None else uniforms
    s = settings(rows, users)
    got, err = run(logits, u, *s)
    want = sampled(logits, u, *s)
    bad = (got != want).nonzero()[:, 0].tolist()
    assert not bad, [(r, users[r % len(users)], float(u[r]), int(got[r]), int(want[r])) for r in bad[:5]]
    return err


def normal(rows, vocab, dtype=F32, scale=3.0, seed=0):
    return (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def peaked(rows, vocab, dtype=F32, seed=0):
    """A few likely columns above the rest."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * 2
    many = min(300, vocab)
    at = torch.randperm(vocab, generator=g)[:many]
    x[:, at] = 17 - 1.7 * torch.log1p(torch.arange(many).float()) + 0.5 * torch.randn(rows, many, generator=g)
    return x.to(dtype)


OFF = (1.0, 0, 1.0, 0.0)
USERS = [OFF, (0.7, 50, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.0, 5, 0.5, 0.1), (0.8, 0, 1.0, 0.05), (1.2, 200, 0.99, 0.01),
         (1.0, 1, 1.0, 0.0), (0.9, 1000, 1.0, 0.0), (1.5, 3, 0.3, 0.5), (0.3, 0, 0.999, 0.0)]  # fmt: skip


@pytest.mark.parametrize("dtype", [F32, BF16, FP16])
@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 33, 255, 1000, 4096, 4097, 8193, 32767, 32769, 50257, 128001])
def test_vocabularies_and_types(vocab, dtype):
    assert check(normal(10, vocab, dtype, seed=vocab), USERS, 1) == 0
    assert check(peaked(10, vocab, dtype, seed=vocab), USERS, 2) == 0


@pytest.mark.parametrize("seed", range(3))
@pytest.mark.parametrize("make", [normal, peaked])
def test_many_rows(make, seed):
    check(make(300, 2003, seed=seed), USERS, seed)


@pytest.mark.parametrize("k", [1, 2, 31, 32, 33, 100, 1023, 1024, 1025, 3000, 20000, 50256, 50257, 60000, -1])
def test_top_k(k):
    check(normal(4, 50257, seed=k), [(1.0, k, 1.0, 0.0)], k + 2)
    check(normal(4, 50257, BF16, seed=k), [(1.0, k, 0.8, 0.0)], k + 2)


@pytest.mark.parametrize("p", [0.0, -1.0, 1e-30, 0.01, 0.5, 0.9, 0.99, 0.9999, 1 - 2.0**-24, 1.0, 2.0, math.inf, math.nan])
@pytest.mark.parametrize("k", [0, 40])
def test_top_p(p, k):
    for make in (normal, peaked):
        check(make(6, 50257, seed=3), [(1.0, k, p, 0.0), (0.6, k, p, 0.0)], 4)
        check(make(6, 5000, FP16, seed=3), [(1.0, k, p, 0.0), (0.6, k, p, 0.0)], 4)


@pytest.mark.parametrize("m", [-0.1, 0.0, 1e-30, 1e-6, 0.01, 0.3, 0.99, 1.0, 7.0, math.nan])
def test_min_p(m):
    check(peaked(6, 50257, seed=5), [(1.0, 0, 1.0, m), (0.7, 30, 0.9, m)], 6)


def test_draws_everywhere():
    # The uniforms walk over the unit interval, and its ends.
    for users in ([OFF], [(1.0, 300, 1.0, 0.0)], [(1.0, 0, 0.7, 0.0)], [(1.0, 0, 1.0, 0.002)]):
        logits = peaked(1, 9001, seed=7).expand(256, 9001).contiguous()
        check(logits, users, uniforms=torch.cat([torch.arange(255) / 255, torch.tensor([1 - 2.0**-24])]))


# ---- equal logits: ranks by column, the lowest first
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [700, 40000])
def test_all_equal(vocab, dtype):
    logits = torch.zeros(8, vocab, dtype=dtype)
    u = torch.tensor([0.0, 0.2, 0.5, 0.9, 0.999, 0.3, 0.6, 0.75])
    for k in (1, 2, 5, 33, 699):
        got, _ = run(logits, u, *settings(8, [(1.0, k, 1.0, 0.0)]))
        assert torch.equal(got, (u.double() * k).floor().long())
    for p in (0.25, 0.5, 0.75):
        got, _ = run(logits, u, *settings(8, [(1.0, 0, p, 0.0)]))
        assert torch.equal(got, (u.double() * math.ceil(p * vocab)).floor().long())
    got, _ = run(logits, u, *settings(8, [(1.0, 8, 0.5, 0.0)]))
    assert torch.equal(got, (u.double() * 4).floor().long())


def test_ties_at_the_cut():
    # Few values: every cut falls among equal logits, spread over all columns.
    for vocab in (500, 33000):
        for dtype in (F32, BF16):
            g = torch.Generator().manual_seed(vocab)
            logits = torch.randint(-3, 4, (40, vocab), generator=g).to(dtype)
            check(logits, [(1.0, k, p, 0.0) for k in (0, 1, 7, 100, 450) for p in (1.0, 0.9, 0.33)], 8)


def test_minus_zero_is_zero():
    logits = torch.zeros(4, 100)
    logits[:, ::2] = -0.0
    u = torch.tensor([0.0, 0.3, 0.6, 0.9])
    got, _ = run(logits, u, *settings(4, [(1.0, 10, 1.0, 0.0)]))
    assert torch.equal(got, (u.double() * 10).floor().long())  # (0.9 in float32 is below 9 / 10: the last is 8)


# ---- masked tokens, rows without a distribution, extreme values
def test_masked_tokens_are_never_drawn():
    for masked in (slice(3000, None), slice(0, 6000)):
        logits = normal(64, 9001, seed=9)
        logits[:, masked] = -math.inf
        check(logits, USERS, 9)
    logits = torch.full((8, 20000), -math.inf)
    logits[:, 19999] = -5.0
    assert check(logits, USERS, 10) == 0


def test_lowest_value_masks():
    for dtype in (F32, BF16, FP16):
        logits = normal(20, 5000, dtype, seed=11)
        logits[:, 40:] = torch.finfo(dtype).min
        assert check(logits, USERS, 11) == 0


def test_rows_without_a_distribution_are_flagged_and_greedy():
    for spoil in (math.nan, math.inf, -math.nan):
        logits = normal(4, 9000, seed=12)
        logits[1, 8500] = spoil
        logits[1, 8700] = spoil
        assert check(logits, [(1.0, 5, 0.9, 0.0)], 12) == _lib.DEVERR_VALUE
        assert int(run(logits, torch.rand(4), torch.ones(4))[0][1]) == 8500
        assert check(logits, [(0.0, 5, 0.9, 0.0)], 12) == 0
    logits[1] = -math.inf
    assert check(logits, [(1.0, 0, 0.9, 0.0)], 12) == _lib.DEVERR_VALUE


def test_extreme_logits_and_temperatures():
    check(normal(10, 9000, seed=13) * 1e30, USERS, 13)
    check(normal(10, 9000, seed=13) * 1e-30, USERS, 13)
    for t in (1e-30, 1e-5, 1e5, 1e30, math.inf):
        check(normal(10, 9000, seed=14), [(t, 0, 1.0, 0.0), (t, 20, 0.9, 0.0), (t, 0, 0.5, 0.0)], 14)
    assert check(normal(10, 900, seed=14), [(math.nan, 0, 1.0, 0.0), (-1.0, 0, 0.5, 0.0)], 14) == 0  # not above 0: greedy


def test_values_far_apart():
    # Columns in every octave below the largest, also negative ones: the cuts lie far from it.
    x = torch.cat([2.0 ** torch.arange(-60, 30.0), -(2.0 ** torch.arange(-60, 30.0)), torch.zeros(3)])
    g = torch.Generator().manual_seed(15)
    logits = x[torch.randperm(x.numel(), generator=g)].expand(40, -1).contiguous()
    check(logits, [(3e8, k, p, 0.0) for k in (0, 3, 60, 93, 95, 150) for p in (1.0, 0.99, 0.6)], 15)


# ---- forms of the call
def test_settings_of_sequences():
    logits, u = normal(20, 3001, seed=16), torch.rand(20)
    cu = torch.tensor([2, 2, 7, 8, 8, 17], dtype=torch.int32)  # empty sequences; rows before and behind
    t, k, p, m = settings(5, USERS[1:])
    tokens = torch.full((20,), -7, dtype=torch.int64, device="cuda")
    got, err = run(logits, u, t, k, p, m, cu_seqlens_q=cu, tokens=tokens)
    owner = torch.repeat_interleave(torch.arange(5), cu.diff().long())
    want = sampled(logits[2:17], u[2:17], t[owner], k[owner], p[owner], m[owner])
    assert torch.equal(got[2:17], want) and err == 0
    assert bool((got[:2] == -7).all()) and bool((got[17:] == -7).all())
    fresh, err = run(logits, u, t, k, p, m, cu_seqlens_q=cu)
    assert torch.equal(fresh[2:17], want) and err == 0
    assert bool((fresh[:2] == -1).all()) and bool((fresh[17:] == -1).all())


def test_many_sequences_and_empty_ones():
    g = torch.Generator().manual_seed(30)
    counts = torch.randint(0, 3, (500,), generator=g)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).int()
    rows = int(cu[-1])
    logits, u = normal(rows, 701, BF16, seed=30), torch.rand(rows, generator=g)
    s = settings(500, USERS)
    owner = torch.repeat_interleave(torch.arange(500), counts)
    got, err = run(logits, u, *s, cu_seqlens_q=cu)
    assert torch.equal(got, sampled(logits, u, *(x[owner] for x in s))) and err == 0


def test_calls_on_two_streams_at_once():
    a, b = peaked(60, 50257, seed=31), normal(60, 50257, BF16, seed=32)
    u, s = torch.rand(60), settings(60, USERS)
    want = [sampled(x, u, *s) for x in (a, b)]
    x = [a.cuda(), b.cuda()]
    args = [u.cuda(), *(v.cuda() for v in s)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.sample_tokens(x[i], *args))
    torch.cuda.synchronize()
    assert all(torch.equal(t.cpu(), want[i]) for i in range(2) for t in got[i])

def test_settings_may_be_left_out():
    logits, u = peaked(12, 5003, seed=17), torch.rand(12)
    t = torch.full((12,), 0.8)
    k, p, m = torch.full((12,), 9, dtype=torch.int32), torch.full((12,), 0.7), torch.full((12,), 0.1)
    for have in range(8):
        args = [x if have >> i & 1 else None for i, x in enumerate((k, p, m))]
        assert torch.equal(run(logits, u, t, *args)[0], sampled(logits, u, t, *args))


def test_strided_rows_and_empty_calls():
    want = normal(9, 5001, BF16, seed=18)
    logits = torch.zeros(9, 5107, dtype=BF16, device="cuda")[:, 7 : 7 + 5001]
    logits.copy_(want)
    u, s = torch.rand(9), settings(9, USERS)
    assert torch.equal(run(logits, u, *s)[0], sampled(want, u, *s))
    assert run(torch.zeros(0, 50), torch.zeros(0), torch.zeros(0))[0].shape == (0,)
    tokens = torch.full((3,), 5, dtype=torch.int64, device="cuda")
    got, _ = run(torch.zeros(3, 50), torch.zeros(3), torch.zeros(0), cu_seqlens_q=torch.zeros(1, dtype=torch.int32), tokens=tokens)
    assert got.tolist() == [5, 5, 5]


def test_greedy_is_argmax_rows():
    logits = normal(33, 50257, seed=19)
    got, _ = run(logits, torch.rand(33), torch.zeros(33))
    assert torch.equal(got, ops.argmax_rows(logits.cuda()).cpu())


def test_the_largest_vocabulary():
    logits = normal(3, 2**21, seed=20)
    check(logits, [OFF, (1.0, 40, 0.9, 0.0), (1.0, 0, 0.9, 0.0)], 20)


def test_streams_and_graphs():
    logits, u = peaked(40, 50257, seed=21).cuda(), torch.rand(40).cuda()
    s = [x.cuda() for x in settings(40, USERS)]
    want = ops.sample_tokens(logits, u, *s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.sample_tokens(logits, u, *s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.sample_tokens(logits, u, *s)
        graphs.append(graph)
        outs.append(out)
    for turn in range(3):
        u.copy_(torch.rand(40, generator=torch.Generator().manual_seed(turn)))
        logits.copy_(logits.roll(turn, 1))
        for graph in graphs:
            graph.replay()
        want = ops.sample_tokens(logits, u, *s)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        assert torch.equal(want.cpu(), sampled(logits.cpu(), u.cpu(), *(x.cpu() for x in s)))


@pytest.mark.parametrize("rows", [96, 160])
def test_draws_that_meet_the_border_of_a_chunk(rows):
    # 16 times the same 2,048 columns, and uniform numbers of whole sixteenths: what lies before the chunk (of 2,048 columns, or of 8,192
    # with many rows) or the round (4,096) that the token falls in is the goal itself, up to roundings to either side. The token is
    # the first column of that sixteenth, or by those roundings the one before. Every weight is far above them.
    g = torch.Generator().manual_seed(33)
    logits = torch.cat([torch.rand(rows, 2048, generator=g) * -3.0] * 16, 1)
    sixteenth = torch.arange(rows) % 16
    for turn, t in enumerate((0.3, 0.7, 1.0, 1.3, 2.7)):
        got, err = run(logits.roll(turn, 0), sixteenth / 16, torch.full((rows,), t))
        off = got - 2048 * sixteenth
        assert err == 0 and bool(((off == 0) | ((off == -1) & (sixteenth > 0))).all()), (t, off.tolist())


@pytest.mark.parametrize("k", [0, 1_500_000])
@pytest.mark.parametrize("octaves", [42.8, 43.2, 44.3])
@pytest.mark.parametrize("p", [1 - 2.0**-23, 1 - 2.0**-24])
def test_top_p_of_a_long_tail_of_tiny_weights(p, octaves, k):
    # One likely column and 2^21 - 1 others that together weigh a few times as much as p leaves out.
    vocab, first, u = 1 << 21, 7, 1 - 2.0**-24
    logits = torch.full((2, vocab), -octaves * math.log(2.0))
    logits[:, first] = 0.0
    w = math.exp(float(logits[0, 0]))
    total = 1 + ((k or vocab) - 1) * w
    kept = max(0, math.ceil((p * total - 1) / w))  # of the tail: those before which less than p of the sum lies
    goal = u * (1 + kept * w)
    want = math.floor((goal - 1) / w)  # of the tail's columns, the one that passes it; below 0: the likely column does
    got, err = run(logits, torch.full((2,), u), torch.ones(2), torch.full((2,), k, dtype=torch.int32), torch.full((2,), p))
    assert err == 0
    # Sums of 2^21 weights in fixed point are off by at most vocab 2^-52 of them; the exponentials (2.2e-12 of the tail) and fp64
    # additions (2^-53 each, 512 rounds of them and the chunks') less than 2^-40 in all.
    slack = (vocab * 2.0**-52 + 2.0**-40) / w + 2
    for column in got.tolist():
        assert abs(column - (column > first) - want) <= slack if goal > 1 else column == first, (column, want, kept, slack)


def test_subnormal_temperatures_and_flat_rows():
    # Temperatures below the normal numbers, and logits that lie as close: a distribution as flat as any other, of which top-p leaves
    # thousands of columns.
    g = torch.Generator().manual_seed(34)
    for vocab in (50257, 9001):
        logits = torch.randint(0, 8_000_000, (12, vocab), generator=g, dtype=torch.int32).view(torch.float32)
        for bits in (30_000, 2_000_000, 6_000_000):
            t = float(torch.tensor([bits], dtype=torch.int32).view(torch.float32))
            check(logits, [(t, 0, 0.9, 0.0), (t, 0, 0.5, 0.0), (t, 0, 1.0, 0.0), (t, 9000, 0.7, 0.0), (t, 20000, 0.3, 0.0)], bits)
