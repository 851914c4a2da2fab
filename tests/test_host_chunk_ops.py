"""rope_cache_write, paged_chunk and verify_drafts without a GPU: schemas, what the operators' fakes and the C ABI refuse
before any launch, workspace sizes, the rotation table."""

from __future__ import annotations

import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from tokquay_amd import _lib, ops, torch_ops

BF16 = torch.bfloat16


def rope_args(dtype=BF16, d=64):
    e = lambda *s, **k: torch.empty(*s, device="cuda", **{"dtype": dtype, **k})  # noqa: E731
    return dict(q_out=e(5, 4, d), q=e(5, 4, d), k=e(5, 2, d), v=e(5, 2 * d), pool=e(8, 2, 2, 2, 16, d), layer=1,
                slot_mapping=e(5, dtype=torch.int64), positions=e(5, dtype=torch.int64),
                table=e(100, d, dtype=torch.float32), interleaved=False, q_norm=e(d), k_norm=e(d), eps=1e-6,
                d_error=e(1, dtype=torch.int32))  # fmt: skip


def chunk_args(dtype=BF16, d=64):
    e = lambda *s, **k: torch.empty(*s, device="cuda", **{"dtype": dtype, **k})  # noqa: E731
    i = dict(dtype=torch.int32)
    return dict(out=e(7, 4 * d), q=e(7, 4, d), pool=e(8, 2, 2, 2, 16, d), layer=0, block_tables=e(3, 4, **i),
                cu_seqlens_q=e(4, **i), q_start=e(3, **i), max_query_len=4, max_context_len=64, scale=0.125,
                workspace=e(4096, dtype=torch.uint8), d_error=e(1, **i))  # fmt: skip


def verify_args():
    e = lambda *s, dtype=torch.float32: torch.empty(*s, device="cuda", dtype=dtype)  # noqa: E731
    return dict(tokens=e(2, 3, dtype=torch.int64), accepted=e(2, dtype=torch.int32), logits=e(5, 90), draft_probs=e(5, 90),
                draft_tokens=e(5, dtype=torch.int64), uniforms=e(5), temperature=e(2), cu_seqlens_q=e(3, dtype=torch.int32),
                d_error=e(1, dtype=torch.int32))  # fmt: skip


ARGS = {"rope_cache_write": rope_args, "paged_chunk": chunk_args, "verify_drafts": verify_args}


def inner_strided(t):
    return torch.empty(*t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype, device=t.device)[..., ::2]


def other_type(t):
    return torch.empty_like(t, dtype=torch.float64)


def host(t):
    return torch.empty(t.shape, dtype=t.dtype, device="cpu")


def shorter(t):
    return t[:-1]


def off_by_four(t):  # the same shape, 4 elements (8 bytes) into its storage
    return torch.empty(t.numel() + 4, dtype=t.dtype, device=t.device)[4:].view(t.shape)


SPOILED = {
    "rope_cache_write": [("q", shorter), ("q_out", shorter), ("k", shorter), ("v", shorter), ("positions", shorter),
                         *((n, f) for n in ("q_out", "q", "k", "v", "pool", "slot_mapping", "positions", "table", "q_norm",
                                            "k_norm") for f in (other_type, host, inner_strided)),
                         ("q", lambda t: t[..., :32]), ("q_out", lambda t: t[:, :2]), ("k", lambda t: t[:, :1]),
                         ("q", off_by_four), ("k_norm", off_by_four), ("layer", lambda v: 2), ("layer", lambda v: -1),
                         ("table", lambda t: t[:, :24].contiguous()), ("d_error", host), ("q_norm", lambda t: t[:32])],
    "paged_chunk": [*((n, f) for n in ("out", "q", "pool", "block_tables", "cu_seqlens_q", "q_start")
                      for f in (other_type, host, inner_strided)), ("out", shorter), ("block_tables", shorter),
                    ("cu_seqlens_q", shorter), ("layer", lambda v: 2), ("max_query_len", lambda v: -1),
                    ("max_context_len", lambda v: 2**31), ("pool", lambda t: t.float()), ("q", lambda t: t.half()),
                    ("q", lambda t: t[:, :3]), ("q", off_by_four), ("workspace", host), ("workspace", inner_strided),
                    ("d_error", host)],
    "verify_drafts": [*((n, f) for n in ("tokens", "accepted", "logits", "draft_probs", "draft_tokens", "uniforms",
                                         "temperature", "cu_seqlens_q") for f in (other_type, host, inner_strided)),
                      ("draft_tokens", shorter), ("uniforms", shorter), ("cu_seqlens_q", shorter), ("tokens", shorter),
                      ("draft_probs", shorter), ("draft_probs", lambda t: t[:, :80]), ("d_error", host)],
}  # fmt: skip
CASES = [(op, name, i) for op, all_ in SPOILED.items() for i, (name, _) in enumerate(all_)]


@pytest.mark.parametrize("op", list(ARGS))
def test_fakes_accept_well_formed_arguments(op):
    with FakeTensorMode():
        getattr(torch_ops.load(), op)(*ARGS[op]().values())


@pytest.mark.parametrize("op,name,i", CASES, ids=lambda v: str(v))
def test_fakes_refuse_spoiled_arguments(op, name, i):
    with FakeTensorMode():
        args = ARGS[op]()
        args[name] = SPOILED[op][i][1](args[name])
        with pytest.raises(RuntimeError, match=f"tokquay_amd::{op}: "):
            getattr(torch_ops.load(), op)(*args.values())


def test_schemas_name_what_is_written():
    ops_ = torch_ops.load()
    written = {"rope_cache_write": ("q_out", "pool"), "paged_chunk": ("out",), "verify_drafts": ("tokens", "accepted")}
    for name, outs in written.items():
        schema = getattr(ops_, name).default._schema
        mutated = {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write}
        assert mutated == set(outs) | {"d_error"} | ({"workspace"} if name == "paged_chunk" else set())


def test_optional_arguments_may_be_left_out():
    with FakeTensorMode():
        a = rope_args()
        ops.rope_cache_write(*[a[n] for n in ("q_out", "q", "k", "v", "pool", "layer", "slot_mapping", "positions", "table")])
        a = chunk_args()
        ops.paged_chunk(*[a[n] for n in ("out", "q", "pool", "layer", "block_tables", "cu_seqlens_q", "q_start",
                                         "max_query_len", "max_context_len")])  # fmt: skip
        a = verify_args()
        tokens, accepted = ops.verify_drafts(a["logits"], a["draft_tokens"], a["uniforms"], a["cu_seqlens_q"], 3, a["temperature"])
        assert tokens.shape == (2, 3) and accepted.shape == (2,)


def test_wrappers_raise_value_errors():
    with FakeTensorMode():
        a = rope_args()
        a["layer"] = 7
        with pytest.raises(ValueError, match="rope_cache_write: layer 7 out of range"):
            ops.rope_cache_write(**a)


def test_a_traced_step_records_the_kernels_as_operators():
    torch_ops.load()

    def step(q_out, q, k, v, pool, slots, positions, table, out, tables, cu, start):
        torch.ops.tokquay_amd.rope_cache_write(q_out, q, k, v, pool, 0, slots, positions, table, False, None, None, 1e-6, None)
        torch.ops.tokquay_amd.paged_chunk(out, q_out, pool, 0, tables, cu, start, 4, 64, 0.125, None, None)
        return out.sum()

    with FakeTensorMode():
        r, c = rope_args(), chunk_args()
        args = [r[n] for n in ("q_out", "q", "k", "v", "pool", "slot_mapping", "positions", "table")]
        out = torch.empty(5, 4, 64, dtype=BF16, device="cuda")
        graph = make_fx(step)(*args, out, c["block_tables"], c["cu_seqlens_q"], c["q_start"])
    targets = [str(n.target) for n in graph.graph.nodes if n.op == "call_function"]
    assert "tokquay_amd.rope_cache_write.default" in targets and "tokquay_amd.paged_chunk.default" in targets


def test_rope_table_is_the_angles_cosines_and_sines():
    t = ops.rope_table(1000, 32, base=1000.0)
    assert t.shape == (1000, 32) and t.dtype == torch.float32
    for p in (0, 1, 999):
        for i in (0, 1, 15):
            a = p * 1000.0 ** (-2 * i / 32)
            assert abs(float(t[p, i]) - math.cos(a)) <= 2.0**-24 and abs(float(t[p, 16 + i]) - math.sin(a)) <= 2.0**-24
    for bad in ((0, 32), (10, 0), (10, 7)):
        with pytest.raises(ValueError):
            ops.rope_table(*bad)


# ---- C ABI: nothing is launched, so the addresses are never used
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3
P = 4096  # an aligned address


def rope_call(q_out=P, qs=256, q=P, k=P, v=P, kvs=128, pool=P, nb=8, layers=2, heads=4, kv=2, bs=16, d=64, layer=0, slots=P,
              pos=P, table=P, positions=100, rotary=64, inter=0, qn=None, kn=None, eps=1e-6, n=5, dtype=2):  # fmt: skip
    return _lib.lib().tq_rope_cache_write(q_out, qs, q, qs, k, kvs, v, kvs, pool, nb, layers, heads, kv, bs, d, layer, slots,
                                          pos, table, positions, rotary, inter, qn, kn, eps, n, dtype, None, None)  # fmt: skip


@pytest.mark.parametrize("status,more", [
    (INVALID, dict(n=-1)), (INVALID, dict(nb=0)), (INVALID, dict(layer=2)), (INVALID, dict(heads=0)), (INVALID, dict(kv=0)),
    (INVALID, dict(bs=0)), (INVALID, dict(rotary=0)), (INVALID, dict(rotary=80)), (INVALID, dict(inter=2)),
    (INVALID, dict(eps=-1.0)), (INVALID, dict(eps=math.nan)), (UNSUPPORTED, dict(d=96)), (UNSUPPORTED, dict(bs=1025)),
    (UNSUPPORTED, dict(rotary=24)), (UNSUPPORTED, dict(nb=1 << 32)), (UNSUPPORTED, dict(n=1 << 32)), (UNSUPPORTED, dict(dtype=3)), (UNSUPPORTED, dict(dtype=-1)), (OK, dict(n=0)),
    (INVALID, dict(q=None)), (INVALID, dict(q_out=None)), (INVALID, dict(pool=None)), (INVALID, dict(slots=None)),
    (INVALID, dict(pos=None)), (INVALID, dict(table=None)), (INVALID, dict(qs=248)), (INVALID, dict(kvs=120)),
    (INVALID, dict(q=P + 8)), (INVALID, dict(table=P + 4)), (INVALID, dict(qn=P + 2)), (INVALID, dict(qs=260)),
])  # fmt: skip
def test_rope_cache_write_c_refusals(status, more):
    assert rope_call(**more) == status


def chunk_call(out=P, os=256, q=P, qs=256, pool=P, nb=8, layers=2, heads=4, kv=2, bs=16, d=64, layer=0, tables=P, ts=4,
               mb=4, cu=P, start=P, seqs=3, rows=7, mq=4, mc=64, scale=0.1, dtype=2, ws=None, wb=0):  # fmt: skip
    return _lib.lib().tq_paged_chunk(out, os, q, qs, pool, nb, layers, heads, kv, bs, d, layer, tables, ts, mb, cu, start,
                                     seqs, rows, mq, mc, scale, dtype, ws, wb, None, None)  # fmt: skip


@pytest.mark.parametrize("status,more", [
    (INVALID, dict(seqs=-1)), (INVALID, dict(rows=-1)), (INVALID, dict(mq=-1)), (INVALID, dict(mc=-1)),
    (INVALID, dict(heads=5)), (INVALID, dict(kv=0)), (INVALID, dict(nb=0)), (INVALID, dict(layer=-1)),
    (INVALID, dict(scale=math.inf)), (INVALID, dict(scale=math.nan)), (UNSUPPORTED, dict(d=96)),
    (UNSUPPORTED, dict(bs=1025)), (UNSUPPORTED, dict(dtype=0)),
    (UNSUPPORTED, dict(mc=(1 << 30) + 1)), (OK, dict(seqs=0)), (OK, dict(rows=0)), (OK, dict(mq=0)),
    (INVALID, dict(out=None)), (INVALID, dict(q=None)), (INVALID, dict(pool=None)), (INVALID, dict(tables=None)),
    (INVALID, dict(cu=None)), (INVALID, dict(start=None)), (INVALID, dict(ts=3)), (INVALID, dict(os=255)),
    (INVALID, dict(qs=248)), (INVALID, dict(mc=0)), (INVALID, dict(q=P + 8)), (INVALID, dict(out=P + 4)),
    (INVALID, dict(qs=260)), (INVALID, dict(os=258)), (WORKSPACE, dict(mc=5000, mb=400, ts=400)),
    (WORKSPACE, dict(mc=5000, mb=400, ts=400, ws=P, wb=16)), (WORKSPACE, dict(mc=5000, mb=400, ts=400, ws=P + 4, wb=1 << 30)),
])  # fmt: skip
def test_paged_chunk_c_refusals(status, more):
    assert chunk_call(**more) == status


def verify_call(tokens=P, accepted=P, logits=P, ls=90, probs=None, ps=90, drafts=P, u=P, temp=P, cu=P, seqs=2, rows=5, mr=3,
                vocab=90, dtype=0, ws=P, wb=1 << 20):  # fmt: skip
    return _lib.lib().tq_verify_drafts(tokens, accepted, logits, ls, probs, ps, drafts, u, temp, cu, seqs, rows, mr, vocab,
                                       dtype, ws, wb, None, None)  # fmt: skip


@pytest.mark.parametrize("status,more", [
    (INVALID, dict(seqs=-1)), (INVALID, dict(rows=-1)), (INVALID, dict(mr=-1)), (INVALID, dict(vocab=0)),
    (UNSUPPORTED, dict(dtype=5)), (UNSUPPORTED, dict(vocab=(1 << 21) + 1)), (OK, dict(seqs=0)), (INVALID, dict(mr=0)),
    (INVALID, dict(tokens=None)), (INVALID, dict(accepted=None)), (INVALID, dict(logits=None)), (INVALID, dict(drafts=None)),
    (INVALID, dict(u=None)), (INVALID, dict(temp=None)), (INVALID, dict(cu=None)), (INVALID, dict(ls=89)),
    (INVALID, dict(probs=P, ps=89)), (WORKSPACE, dict(ws=None)), (WORKSPACE, dict(wb=8)), (WORKSPACE, dict(ws=P + 8)),
])  # fmt: skip
def test_verify_drafts_c_refusals(status, more):
    assert verify_call(**more) == status


def test_workspace_sizes():
    size = ops.chunk_workspace_bytes
    assert size(128, 32, 8, 128, 128, 1, 100) == 0  # the rows fill the GPU
    assert size(1, 32, 8, 128, 1, 1, 64) == 0  # one step of keys
    long = size(1, 32, 8, 128, 1, 1, 4000)
    assert long > 0 and long % ((128 + 2) * 4 * 32) == 0
    assert size(0, 32, 8, 128, 0, 0, 0) == 0 and size(1, 32, 7, 128, 1, 1, 4000) == 0
    assert _lib.lib().tq_verify_drafts_workspace_size(2, 10, 50257) > _lib.lib().tq_verify_drafts_workspace_size(2, 5, 50257) > 0
    assert _lib.lib().tq_verify_drafts_workspace_size(0, 0, 50257) == 0


# What depends on values rather than tensors: the fakes refuse it as the operators do.
UNFIT = {
    "rope_cache_write": [("eps", -1.0), ("eps", math.nan), ("table", lambda t: t[:0]),
                         ("pool", lambda t: t.new_empty(1 << 23, 1, 2, 2, 1024, 64)), ("tokens", 1 << 30)],
    "paged_chunk": [("scale", math.inf), ("scale", -math.inf), ("scale", math.nan), ("scale", 1e300), ("max_context_len", (1 << 30) + 1),
                    ("max_context_len", 0), ("max_query_len", 1 << 30), ("block_tables", lambda t: t[:, :0]),
                    ("pool", lambda t: t.new_empty(1, 1 << 14, 2, 2, 1024, 64)),
                    ("pool", lambda t: t.new_empty(1 << 31, 1, 2, 2, 1, 64))],
    "verify_drafts": [("rows", 1 << 31), ("tokens", lambda t: t.new_empty(2, 1 << 31))],
}  # fmt: skip


@pytest.mark.parametrize("op,name,i", [(op, name, i) for op, all_ in UNFIT.items() for i, (name, _) in enumerate(all_)],
                         ids=lambda v: str(v))  # fmt: skip
def test_fakes_refuse_unfit_values(op, name, i):
    with FakeTensorMode():
        args, value = ARGS[op](), UNFIT[op][i][1]
        more = lambda t, n: t.new_empty(n, *t.shape[1:])  # noqa: E731
        if op == "rope_cache_write":
            args["layer"] = 0
        if name in ("tokens", "rows") and not callable(value):
            for n in {"tokens": ("q_out", "q", "k", "v", "slot_mapping", "positions"),
                      "rows": ("logits", "draft_probs", "draft_tokens", "uniforms")}[name]:  # fmt: skip
                args[n] = more(args[n], value)
        else:
            args[name] = value(args[name]) if callable(value) else value
        with pytest.raises(RuntimeError, match=f"tokquay_amd::{op}: "):
            getattr(torch_ops.load(), op)(*args.values())


def test_fakes_refuse_short_workspaces():
    with FakeTensorMode():
        args = chunk_args()
        args["max_context_len"], args["block_tables"] = 4000, torch.empty(3, 400, dtype=torch.int32, device="cuda")
        need = ops.chunk_workspace_bytes(3, 4, 2, 64, 7, 4, 4000)
        for bad in (torch.empty(need - 1, dtype=torch.uint8, device="cuda"), torch.empty(need + 8, dtype=torch.uint8, device="cuda")[8:]):
            args["workspace"] = bad
            with pytest.raises(RuntimeError, match="tq_paged_chunk failed: workspace"):
                torch_ops.load().paged_chunk(*args.values())
            with pytest.raises(_lib.KernelError, match="tq_paged_chunk failed: workspace"):
                ops.paged_chunk(**args)
        args["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        ops.paged_chunk(**args)


def test_calls_without_work_need_no_lengths():
    with FakeTensorMode():
        args = chunk_args()
        ops.paged_chunk(**{**args, "max_query_len": 0, "max_context_len": 0, "block_tables": args["block_tables"][:, :0]})
        args = rope_args()
        for n in ("q_out", "q", "k", "v", "slot_mapping", "positions", "table"):
            args[n] = args[n][:0]
        ops.rope_cache_write(**args)
