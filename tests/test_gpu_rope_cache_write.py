"""rope_cache_write against norm and rotation in float64: types, head layouts, rotated widths, strides, padded rows,
errors, graphs. Tolerances are rotation_bound's; values are copied bit for bit."""

from __future__ import annotations

import math

import pytest
import torch

from tests.chunk_cases import LAYER, rotated, rotation_bound
from tokquay_amd import _lib, ops

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


class Case:
    def __init__(self, tokens, heads, kv_heads, dim, dtype, rotary, interleaved=False, norm=False, block_size=16,
                 padded=0, seed=0):  # fmt: skip
        g = torch.Generator().manual_seed(seed)
        blocks = tokens // block_size + 4
        self.interleaved, self.bs, self.dtype = interleaved, block_size, dtype
        self.q, self.k, self.v = (torch.randn(tokens, h, dim, generator=g).to(dtype) for h in (heads, kv_heads, kv_heads))
        self.pool = torch.randn(blocks, 2, 2, kv_heads, block_size, dim, generator=g).to(dtype)
        self.slots = torch.randperm(blocks * block_size, generator=g)[:tokens]
        self.slots[torch.randperm(tokens, generator=g)[:padded]] = -1
        self.positions = torch.randint(0, 500, (tokens,), generator=g)
        self.table = ops.rope_table(500, rotary)
        self.q_norm, self.k_norm = ((torch.rand(dim, generator=g) + 0.5).to(dtype) if norm else None for _ in range(2))

    def args(self, **more):
        cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
        return {**dict(q_out=torch.full_like(self.q, 7.0, device="cuda"), q=self.q.cuda(), k=self.k.cuda(), v=self.v.cuda(),
                       pool=self.pool.cuda(), layer=LAYER, slot_mapping=self.slots.cuda(), positions=self.positions.cuda(),
                       table=self.table.cuda(), interleaved=self.interleaved, q_norm=cuda(self.q_norm),
                       k_norm=cuda(self.k_norm)), **more}  # fmt: skip

    def check(self, q_out, pool, skipped=()):
        """``skipped``: tokens that write nothing."""
        keep = torch.ones(len(self.slots), dtype=torch.bool)
        keep[list(skipped)] = False
        for got, x, w, rows in ((q_out.cpu(), self.q, self.q_norm, keep), (None, self.k, self.k_norm, keep & (self.slots >= 0))):
            positions = torch.where(keep, self.positions, 0)
            y, size = rotated(x, self.table, positions, self.interleaved, w, 1e-6)
            if got is None:
                at = self.slots[rows]
                got, y, size = pool.cpu()[at // self.bs, LAYER, 0, :, at % self.bs], y[rows], size[rows]
            else:
                got, y, size = got.view(y.shape)[rows], y[rows], size[rows]
            off = (got.double() - y).abs() - rotation_bound(y, size, self.dtype)
            assert bool((off <= 0).all()), float(off.max())
        want = self.pool.clone()
        at = self.slots[keep & (self.slots >= 0)]
        want[at // self.bs, LAYER, 1, :, at % self.bs] = self.v[keep & (self.slots >= 0)]
        want[at // self.bs, LAYER, 0, :, at % self.bs] = pool.cpu()[at // self.bs, LAYER, 0, :, at % self.bs]
        assert torch.equal(pool.cpu(), want)  # values bit for bit, nothing else touched


def run(c, **more):
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    a = c.args(d_error=err, **more)
    ops.rope_cache_write(**a)
    return a["q_out"], a["pool"], int(err)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (64, 16), (64, 48), (128, 128), (128, 32), (128, 112)])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_types_and_rotated_widths(dtype, dim, rotary, interleaved, norm):
    c = Case(37, 6, 2, dim, dtype, rotary, interleaved, norm, padded=5, seed=1)
    q, pool, err = run(c)
    c.check(q, pool)
    assert err == 0


@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (1, 32, 8), (3, 5, 3), (257, 12, 12), (64, 40, 1), (1000, 7, 2)])
@pytest.mark.parametrize("dim", [64, 128])
def test_head_layouts_and_row_counts(tokens, heads, kv_heads, dim):
    c = Case(tokens, heads, kv_heads, dim, BF16, dim, norm=True, block_size=8, seed=2)
    q, pool, err = run(c)
    c.check(q, pool)
    assert err == 0


@pytest.mark.parametrize("block_size", [1, 3, 64, 1024])
def test_block_sizes(block_size):
    c = Case(50, 4, 2, 64, FP16, 64, block_size=block_size, padded=4, seed=3)
    q, pool, _ = run(c)
    c.check(q, pool)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (FP32, 64)])
def test_views_of_a_fused_projection_and_in_place(dtype, dim):
    c = Case(41, 4, 2, dim, dtype, dim, norm=True, seed=4)
    w = torch.randn(41, 8 * dim + 8, device="cuda").to(dtype)
    q, k, v = w[:, : 4 * dim], w[:, 4 * dim : 6 * dim], w[:, 6 * dim : 8 * dim]
    for t, x in ((q, c.q), (k, c.k), (v, c.v)):
        t.copy_(x.view(41, -1))
    before = w.clone()
    _, pool, _ = run(c, q=q, k=k.view(41, 2, dim), v=v, q_out=q)  # the queries in place
    c.check(q.reshape(41, 4, dim), pool)
    assert torch.equal(w[:, 4 * dim :], before[:, 4 * dim :])


def test_only_queries_or_only_keys_normed():
    for drop in ("q_norm", "k_norm"):
        c = Case(20, 4, 2, 128, BF16, 64, norm=True, seed=5)
        setattr(c, drop, None)
        q, pool, _ = run(c)
        c.check(q, pool)


def test_every_row_padded_and_no_rows():
    c = Case(9, 4, 2, 64, BF16, 64, padded=9, seed=6)
    q, pool, err = run(c)
    c.check(q, pool)
    assert torch.equal(pool.cpu(), c.pool) and err == 0
    c = Case(0, 4, 2, 64, BF16, 64, seed=6)
    _, pool, err = run(c)
    assert torch.equal(pool.cpu(), c.pool) and err == 0


def test_values_keep_their_bits():
    c = Case(8, 2, 2, 64, BF16, 64, seed=7)
    c.v = torch.randint(-(2**15), 2**15, c.v.shape).to(torch.int16).view(BF16)  # NaNs with payloads among them
    _, pool, _ = run(c)
    at = c.slots
    assert torch.equal(pool.cpu()[at // c.bs, LAYER, 1, :, at % c.bs].view(torch.int16), c.v.view(torch.int16))


def test_large_and_tiny_heads_keep_fp32_norms():
    c = Case(6, 2, 2, 128, BF16, 128, norm=True, seed=8)
    c.q[0] *= 2.0**40
    c.q[1] *= 2.0**-30
    c.k[2] = 0
    q, pool, _ = run(c)
    c.check(q, pool)


def test_far_positions():
    c = Case(16, 2, 2, 64, FP32, 64, seed=9)
    c.table = ops.rope_table(131072, 64, base=500000.0)
    c.positions = torch.arange(16) * 8191 + 8000
    q, pool, _ = run(c)
    c.check(q, pool)
    i = torch.arange(32, dtype=torch.float64)  # the table's own angles
    want = (c.positions[-1].double() * 500000.0 ** (-i / 32)).cos()
    torch.testing.assert_close(c.table[c.positions[-1], :32].double(), want, rtol=0, atol=2.0**-24)


def test_errors_are_flagged_and_their_rows_skipped():
    c = Case(12, 4, 2, 64, BF16, 64, seed=10)
    c.positions[3] = 500
    c.positions[4] = -1
    q, pool, err = run(c)
    assert err == _lib.DEVERR_POSITION
    c.check(q, pool, skipped=(3, 4))
    assert bool((q[3:5] == 7.0).all())
    c = Case(12, 4, 2, 64, BF16, 64, seed=10)
    c.slots[5] = c.pool.size(0) * 16
    q, pool, err = run(c)
    assert err == _lib.DEVERR_SLOT
    c.slots[5] = -1  # its queries are written, its cache entry is not
    c.check(q, pool)


def test_a_captured_call_replays():
    c = Case(20, 4, 2, 128, BF16, 128, norm=True, seed=11)
    a = c.args()
    ops.rope_cache_write(**a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rope_cache_write(**a)
    for seed in (12, 13):
        c = Case(20, 4, 2, 128, BF16, 128, norm=True, seed=seed)
        for name, t in c.args().items():
            if isinstance(t, torch.Tensor):
                a[name].copy_(t)
        graph.replay()
        c.check(a["q_out"], a["pool"])


def test_a_pool_past_2_31_elements():
    c = Case(5, 2, 1, 128, BF16, 128, block_size=1024, seed=14)
    blocks = 2**31 // (1024 * 128 * 4) + 9
    pool = torch.zeros(blocks, 2, 2, 1, 1024, 128, dtype=BF16, device="cuda")
    far = blocks - c.pool.size(0)
    pool[far:] = c.pool.cuda()
    q, _, err = run(c, pool=pool, slot_mapping=(c.slots + far * 1024).cuda())
    assert err == 0 and not bool(pool[:far].any())
    c.check(q, pool[far:])


def test_refusals():
    c = Case(12, 4, 2, 64, BF16, 64, norm=True, seed=15)
    good = c.args()
    ops.rope_cache_write(**good)
    wide = torch.zeros(12, 4 * 64 + 4, dtype=BF16, device="cuda")
    for name, value in [("q", c.q.cuda().half()), ("q", c.q.cuda()[:-1]), ("q", wide[:, 4:]), ("q_out", good["q_out"][:, :3]),
                        ("k", c.k.cuda()[:, :1]), ("v", c.v.cuda().float()), ("pool", c.pool.cuda().double()),
                        ("pool", c.pool.cuda()[..., :32].contiguous()), ("layer", -1), ("slot_mapping", c.slots.cuda().int()),
                        ("positions", c.positions.cuda()[:-1]), ("table", c.table.cuda().double()),
                        ("table", c.table.cuda()[:, :24].contiguous()), ("q_norm", c.q_norm.cuda().float()),
                        ("k_norm", c.k_norm.cuda()[:32]), ("eps", -1.0), ("eps", math.nan)]:  # fmt: skip
        with pytest.raises((ValueError, _lib.KernelError), match="rope_cache_write"):
            ops.rope_cache_write(**{**good, name: value})


def test_refusals_of_values():
    c = Case(12, 4, 2, 64, BF16, 64, norm=True, seed=15)
    good = c.args()
    for name, value in [("eps", -1.0), ("eps", math.nan), ("table", c.table.cuda()[:0])]:
        with pytest.raises(ValueError, match="rope_cache_write"):
            ops.rope_cache_write(**{**good, name: value})
    none = {n: good[n][:0] for n in ("q_out", "q", "k", "v", "slot_mapping", "positions", "table")}
    ops.rope_cache_write(**{**good, **none})
