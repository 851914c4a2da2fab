"""tree_layout, paged_tree, sample_tokens, accept_tree and copy_blocks without a GPU: schemas, what the operators' fakes and the C ABI
refuse before any launch."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from tests.test_host_chunk_ops import chunk_args, chunk_call, host, inner_strided, off_by_four, other_type, shorter, verify_call
from tokquay_amd import _lib, ops, torch_ops

BF16, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


def empty(*shape, dtype=F32):
    return torch.empty(*shape, device="cuda", dtype=dtype)


def layout_args():
    return dict(positions=empty(70, dtype=I64), masks=empty(70, 2, dtype=I64), parents=empty(70, dtype=I32),
                cu_seqlens_q=empty(4, dtype=I32), q_start=empty(3, dtype=I32), max_query_len=66,
                d_error=empty(1, dtype=I32))  # fmt: skip


def tree_args():
    a = chunk_args()
    out = {}
    for name, value in a.items():
        out[name] = value
        if name == "q_start":
            out["masks"] = empty(7, 1, dtype=I64)
    return out


def sample_args():
    return dict(tokens=empty(5, dtype=I64), logits=empty(5, 90), uniforms=empty(5), temperature=empty(2), top_k=empty(2, dtype=I32),
                top_p=empty(2), min_p=empty(2), cu_seqlens_q=empty(3, dtype=I32), d_error=empty(1, dtype=I32))  # fmt: skip


def accept_args():
    return dict(tokens=empty(3, 6, dtype=I64), path=empty(3, 6, dtype=I32), counts=empty(3, dtype=I32), sampled=empty(20, dtype=I64),
                draft_tokens=empty(20, dtype=I64), parents=empty(20, dtype=I32), cu_seqlens_q=empty(4, dtype=I32),
                pool=empty(8, 2, 2, 2, 16, 64, dtype=BF16), block_tables=empty(3, 4, dtype=I32), q_start=empty(3, dtype=I32),
                d_error=empty(1, dtype=I32))  # fmt: skip


def copy_args():
    return dict(pool=empty(8, 2, 2, 2, 16, 64, dtype=BF16), src_blocks=empty(3, dtype=I32), dst_blocks=empty(3, dtype=I32),
                num_slots=empty(3, dtype=I32), d_error=empty(1, dtype=I32))  # fmt: skip


ARGS = {"tree_layout": layout_args, "paged_tree": tree_args, "sample_tokens": sample_args, "accept_tree": accept_args,
        "copy_blocks": copy_args}  # fmt: skip


def longer(t):
    return t.new_empty(t.size(0) + 1, *t.shape[1:])


def all_of(*names):
    return [(n, f) for n in names for f in (other_type, host, inner_strided, shorter, longer)]


SPOILED = {
    "tree_layout": [*all_of("positions", "masks", "cu_seqlens_q"), ("parents", other_type), ("parents", host), ("parents", inner_strided),
                    ("q_start", other_type), ("q_start", host), ("masks", lambda t: t[:, :1].contiguous()),
                    ("max_query_len", lambda v: 129), ("max_query_len", lambda v: -1), ("d_error", host), ("d_error", other_type)],
    "paged_tree": [*((n, f) for n in ("out", "q", "pool", "block_tables", "cu_seqlens_q", "q_start", "masks")
                     for f in (other_type, host, inner_strided)), ("masks", shorter), ("masks", longer), ("out", shorter),
                   ("masks", lambda t: t[:, :0]), ("max_query_len", lambda v: 65), ("layer", lambda v: 2), ("q", off_by_four),
                   ("cu_seqlens_q", shorter), ("block_tables", shorter), ("workspace", host), ("d_error", host)],
    "sample_tokens": [*all_of("tokens", "uniforms", "top_k", "top_p", "min_p", "cu_seqlens_q"), ("temperature", other_type),
                      ("temperature", host), ("temperature", inner_strided), ("logits", other_type), ("logits", host),
                      ("logits", inner_strided), ("logits", lambda t: t[:, :0]), ("logits", lambda t: t[:1].expand(5, 90)),
                      ("logits", lambda t: t[0]), ("cu_seqlens_q", lambda t: None), ("d_error", host)],
    "accept_tree": [*all_of("tokens", "path", "draft_tokens", "parents", "cu_seqlens_q", "q_start"), ("sampled", other_type),
                    ("sampled", host), ("sampled", shorter), ("counts", other_type), ("counts", longer), ("counts", host),
                    ("tokens", lambda t: t[:, :0]), ("path", lambda t: t[:, :5].contiguous()), ("pool", other_type), ("pool", host),
                    ("pool", inner_strided), ("pool", lambda t: None), ("block_tables", lambda t: None), ("q_start", lambda t: None),
                    ("block_tables", other_type), ("block_tables", shorter), ("block_tables", inner_strided), ("block_tables", host),
                    ("pool", lambda t: t[..., :32].contiguous()), ("pool", off_by_four), ("d_error", host)],
    "copy_blocks": [*all_of("dst_blocks", "num_slots"), ("src_blocks", other_type), ("src_blocks", host), ("src_blocks", inner_strided),
                    ("pool", other_type), ("pool", host), ("pool", inner_strided), ("pool", lambda t: t[..., :32].contiguous()),
                    ("pool", off_by_four), ("pool", lambda t: t[:0]), ("d_error", host), ("d_error", longer)],
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
    written = {"tree_layout": {"positions", "masks"}, "paged_tree": {"out", "workspace"}, "sample_tokens": {"tokens"},
               "accept_tree": {"tokens", "path", "counts", "pool"}, "copy_blocks": {"pool"}}  # fmt: skip
    for name, outs in written.items():
        schema = getattr(torch_ops.load(), name).default._schema
        mutated = {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write}
        assert mutated == outs | {"d_error"}


def test_optional_arguments_may_be_left_out():
    with FakeTensorMode():
        a = layout_args()
        positions, masks = ops.tree_layout(a["parents"], a["cu_seqlens_q"], a["q_start"], 66)
        assert positions.shape == (70,) and masks.shape == (70, 2) and masks.dtype == I64
        a = tree_args()
        ops.paged_tree(*[a[n] for n in ("out", "q", "pool", "layer", "block_tables", "cu_seqlens_q", "q_start", "masks",
                                        "max_query_len", "max_context_len")])  # fmt: skip
        a = sample_args()
        assert ops.sample_tokens(a["logits"], a["uniforms"], empty(5)).shape == (5,)
        a = accept_args()
        tokens, path, counts = ops.accept_tree(a["sampled"], a["draft_tokens"], a["parents"], a["cu_seqlens_q"], 6)
        assert tokens.shape == (3, 6) and path.shape == (3, 6) and counts.shape == (3,) and path.dtype == I32
        a = copy_args()
        ops.copy_blocks(a["pool"], a["src_blocks"], a["dst_blocks"])


def test_wrappers_raise_value_errors():
    with FakeTensorMode():
        a = tree_args()
        with pytest.raises(ValueError, match="paged_tree: masks must be"):
            ops.paged_tree(**{**a, "masks": a["masks"].int()})
        a = sample_args()
        with pytest.raises(ValueError, match="sample_tokens: top_k must be"):
            ops.sample_tokens(a["logits"], a["uniforms"], empty(5), top_k=empty(5))
        a = accept_args()
        with pytest.raises(ValueError, match="go together"):
            ops.accept_tree(a["sampled"], a["draft_tokens"], a["parents"], a["cu_seqlens_q"], 6, pool=a["pool"])
        with pytest.raises(ValueError, match="tokens must be"):
            ops.accept_tree(a["sampled"], a["draft_tokens"], a["parents"], a["cu_seqlens_q"], 5, tokens=a["tokens"])
        with pytest.raises(ValueError, match="max_path be a length above 0"):
            ops.accept_tree(a["sampled"], a["draft_tokens"], a["parents"], a["cu_seqlens_q"], 0)
        with pytest.raises(ValueError, match="accept_tree: parents must be"):
            ops.accept_tree(a["sampled"], a["draft_tokens"], a["parents"][:-1], a["cu_seqlens_q"], 4)
        with pytest.raises(ValueError, match="tree_layout: max_query_len must be a length"):
            ops.tree_layout(empty(5, dtype=I32), empty(2, dtype=I32), empty(1, dtype=I32), -1)
        with pytest.raises(ValueError, match="sample_tokens: uniforms must be"):
            ops.sample_tokens(empty(5, 90), empty(4), empty(5))
        with pytest.raises(ValueError, match="copy_blocks: dst_blocks must be"):
            ops.copy_blocks(copy_args()["pool"], empty(3, dtype=I32), empty(2, dtype=I32))
        with pytest.raises(ValueError, match="tree_layout: masks must be"):
            ops.tree_layout(empty(5, dtype=I32), empty(2, dtype=I32), empty(1, dtype=I32), 70, masks=empty(5, 1, dtype=I64))


def test_a_traced_step_records_the_kernels_as_operators():
    torch_ops.load()

    def step(out, q, pool, tables, cu, start, parents, logits, u, t, drafts):
        positions, masks = ops.tree_layout(parents, cu, start, 4)
        ops.paged_tree(out, q, pool, 0, tables, cu, start, masks, 4, 64)
        tokens = ops.sample_tokens(logits, u, t, cu_seqlens_q=cu)
        ops.copy_blocks(pool, parents, parents)
        return ops.accept_tree(tokens, drafts, parents, cu, 4, pool, tables, start)

    with FakeTensorMode():
        c = chunk_args()
        graph = make_fx(step)(empty(7, 256, dtype=BF16), c["q"], c["pool"], c["block_tables"], c["cu_seqlens_q"], c["q_start"],
                              empty(7, dtype=I32), empty(7, 50), empty(7), empty(3), empty(7, dtype=I64))  # fmt: skip
    targets = [str(n.target) for n in graph.graph.nodes if n.op == "call_function"]
    assert all(any(f"tokquay_amd.{op}.{form}" in targets for form in ("default", "new")) for op in ARGS)


def test_calls_without_work():
    with FakeTensorMode():
        none = empty(0, dtype=I32)
        ops.tree_layout(none, empty(1, dtype=I32), none, 0)
        ops.sample_tokens(empty(0, 5), empty(0), empty(0))
        ops.copy_blocks(copy_args()["pool"], none, none)
        ops.accept_tree(empty(0, dtype=I64), empty(0, dtype=I64), none, empty(1, dtype=I32), 3)


# ---- C ABI: nothing is launched, so the addresses are never used
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3
P = 4096  # an aligned address


def layout_call(positions=P, masks=P, words=2, parents=P, cu=P, start=P, seqs=3, rows=70, mq=66):
    return _lib.lib().tq_tree_layout(positions, masks, words, parents, cu, start, seqs, rows, mq, None, None)


@pytest.mark.parametrize("status,more", [
    (INVALID, dict(seqs=-1)), (INVALID, dict(rows=-1)), (INVALID, dict(mq=-1)), (INVALID, dict(words=-1)), (INVALID, dict(mq=129)),
    (INVALID, dict(words=1 << 40)), (INVALID, dict(positions=None)), (INVALID, dict(masks=None)), (INVALID, dict(parents=None)),
    (INVALID, dict(cu=None)), (INVALID, dict(start=None)), (UNSUPPORTED, dict(seqs=2**31 - 1)), (OK, dict(rows=0)),
])  # fmt: skip
def test_tree_layout_c_refusals(status, more):
    assert layout_call(**more) == status


def tree_call(out=P, os=256, q=P, qs=256, pool=P, nb=8, layers=2, heads=4, kv=2, bs=16, d=64, layer=0, tables=P, ts=4, mb=4, cu=P,
              start=P, masks=P, words=1, seqs=3, rows=7, mq=4, mc=64, scale=0.1, dtype=2, ws=None, wb=0):  # fmt: skip
    return _lib.lib().tq_paged_tree(out, os, q, qs, pool, nb, layers, heads, kv, bs, d, layer, tables, ts, mb, cu, start, masks,
                                    words, seqs, rows, mq, mc, scale, dtype, ws, wb, None, None)  # fmt: skip


@pytest.mark.parametrize("status,more", [
    (INVALID, dict(masks=None)), (INVALID, dict(words=0)), (INVALID, dict(mq=65)), (INVALID, dict(words=1 << 40)),
    (INVALID, dict(words=-1)), (INVALID, dict(heads=5)), (INVALID, dict(layer=2)), (UNSUPPORTED, dict(d=96)),
    (UNSUPPORTED, dict(dtype=0)), (OK, dict(seqs=0)), (OK, dict(rows=0)), (OK, dict(mq=0)), (INVALID, dict(q=P + 8)),
    (WORKSPACE, dict(mc=5000, mb=400, ts=400)), (WORKSPACE, dict(mc=5000, mb=400, ts=400, ws=P, wb=16)),
])  # fmt: skip
def test_paged_tree_c_refusals(status, more):
    assert tree_call(**more) == status


def accept_call(tokens=P, path=P, counts=P, mp=6, sampled=P, drafts=P, parents=P, cu=P, seqs=3, rows=20, pool=P, nb=8, layers=2,
                kv=2, bs=16, d=64, dtype=2, tables=P, ts=4, mb=4, start=P):  # fmt: skip
    return _lib.lib().tq_accept_tree(tokens, path, counts, mp, sampled, drafts, parents, cu, seqs, rows, pool, nb, layers, kv, bs, d,
                                     dtype, tables, ts, mb, start, None, None)  # fmt: skip


@pytest.mark.parametrize("status,more", [
    (INVALID, dict(seqs=-1)), (INVALID, dict(rows=-1)), (INVALID, dict(mp=-1)), (INVALID, dict(mp=0)), (OK, dict(seqs=0)),
    (INVALID, dict(tokens=None)), (INVALID, dict(path=None)), (INVALID, dict(counts=None)), (INVALID, dict(sampled=None)),
    (INVALID, dict(drafts=None)), (INVALID, dict(parents=None)), (INVALID, dict(cu=None)), (INVALID, dict(tables=None)),
    (INVALID, dict(start=None)), (INVALID, dict(nb=0)), (INVALID, dict(nb=1 << 31)), (INVALID, dict(layers=0)), (INVALID, dict(kv=0)),
    (INVALID, dict(bs=0)), (INVALID, dict(mb=-1)), (INVALID, dict(ts=3)), (INVALID, dict(pool=P + 8)), (UNSUPPORTED, dict(d=96)),
    (UNSUPPORTED, dict(bs=1025)), (UNSUPPORTED, dict(dtype=3)), (UNSUPPORTED, dict(layers=1 << 30, kv=1 << 10)),
])  # fmt: skip
def test_accept_tree_c_refusals(status, more):
    assert accept_call(**more) == status


def copy_call(pool=P, nb=8, layers=2, kv=2, bs=16, d=64, dtype=2, src=P, dst=P, slots=None, pairs=3):
    return _lib.lib().tq_copy_blocks(pool, nb, layers, kv, bs, d, dtype, src, dst, slots, pairs, None, None)


def test_copy_blocks_takes_at_most_2_20_pairs():
    assert copy_call(pairs=(1 << 20) + 1) == UNSUPPORTED and copy_call(pairs=2**31 - 1) == UNSUPPORTED
    with FakeTensorMode():
        ids = empty((1 << 20) + 1, dtype=I32)
        with pytest.raises(ValueError, match="more than 1048576"):
            ops.copy_blocks(copy_args()["pool"], ids, ids)
        ops.copy_blocks(copy_args()["pool"], ids[1:], ids[1:])


@pytest.mark.parametrize("status,more", [
    (INVALID, dict(pairs=-1)), (INVALID, dict(nb=0)), (INVALID, dict(nb=1 << 31)), (INVALID, dict(layers=0)), (INVALID, dict(kv=0)),
    (INVALID, dict(bs=0)), (OK, dict(pairs=0)), (INVALID, dict(pool=None)), (INVALID, dict(src=None)), (INVALID, dict(dst=None)),
    (INVALID, dict(pool=P + 8)), (UNSUPPORTED, dict(d=96)), (UNSUPPORTED, dict(bs=1025)), (UNSUPPORTED, dict(dtype=3)),
    (UNSUPPORTED, dict(layers=1 << 30, kv=1 << 10)),
])  # fmt: skip
def test_copy_blocks_c_refusals(status, more):
    assert copy_call(**more) == status


def sample_call(tokens=P, logits=P, ls=90, u=P, t=P, k=P, p=P, m=P, cu=None, seqs=5, rows=5, vocab=90, dtype=0, ws=P, wb=1 << 20):
    return _lib.lib().tq_sample_tokens(tokens, logits, ls, u, t, k, p, m, cu, seqs, rows, vocab, dtype, ws, wb, None, None)


@pytest.mark.parametrize("status,more", [
    (INVALID, dict(seqs=-1)), (INVALID, dict(rows=-1)), (INVALID, dict(vocab=0)), (UNSUPPORTED, dict(vocab=(1 << 21) + 1)),
    (UNSUPPORTED, dict(dtype=3)), (OK, dict(rows=0)), (INVALID, dict(tokens=None)), (INVALID, dict(logits=None)),
    (INVALID, dict(u=None)), (INVALID, dict(t=None)), (INVALID, dict(seqs=4)), (INVALID, dict(ls=89)), (OK, dict(seqs=0, cu=P)),
    (WORKSPACE, dict(ws=None)), (WORKSPACE, dict(wb=8)), (WORKSPACE, dict(ws=P + 8)),
])  # fmt: skip
def test_sample_tokens_c_refusals(status, more):
    assert sample_call(**more) == status


# ---- more workgroups than a launch takes: 2^32 - 1 threads
GIB = dict(nb=300, layers=16, kv=64, bs=1024, d=128, dtype=0)  # blocks of 1 GiB


@pytest.mark.parametrize("call,more", [
    (layout_call, dict(seqs=2**23 - 1, mq=449, words=8)), (layout_call, dict(seqs=2**26)), (accept_call, dict(seqs=2**24, pool=None)),
    (accept_call, dict(seqs=2**18, layers=64, kv=64, d=64)), (accept_call, dict(seqs=2**30)), (copy_call, dict(GIB, pairs=128)),
    (copy_call, dict(GIB, pairs=256)), (sample_call, dict(rows=2**22, seqs=2**22, wb=1 << 40)),
    (sample_call, dict(rows=2**16, seqs=2**16, vocab=1 << 21, ls=1 << 21, wb=1 << 60)),
    (sample_call, dict(rows=2**31 - 1, seqs=2**31 - 1, wb=1 << 60)), (sample_call, dict(rows=2**22, seqs=1, cu=P, wb=1 << 40)),
    (tree_call, dict(seqs=2**26, rows=2**30)), (tree_call, dict(seqs=2**23, rows=2**30, heads=12, kv=3, qs=768, os=768)),
    (chunk_call, dict(seqs=2**26, rows=2**30)), (verify_call, dict(rows=2**24, seqs=2**20, wb=1 << 60)),
    (verify_call, dict(rows=2**22, seqs=2**22, wb=1 << 60)), (verify_call, dict(rows=2**24, seqs=2**24, probs=P, wb=1 << 60)),
])  # fmt: skip
def test_launches_that_are_too_large_are_refused(call, more):
    assert call(**more) == UNSUPPORTED


def test_fakes_refuse_launches_that_are_too_large():
    with FakeTensorMode():
        with pytest.raises(ValueError, match="tree_layout: q_start has too many sequences"):
            ops.tree_layout(empty(5, dtype=I32), empty(2**23, dtype=I32), empty(2**23 - 1, dtype=I32), 449)
        with pytest.raises(ValueError, match="sample_tokens: logits has too many rows"):
            ops.sample_tokens(empty(2**22, 50), empty(2**22), empty(2**22))
        with pytest.raises(ValueError, match="sample_tokens: logits has too many rows"):
            ops.sample_tokens(empty(2**16, 2**21), empty(2**16), empty(2**16))
        ids = empty(5, dtype=I64)
        with pytest.raises(ValueError, match="accept_tree: counts has too many sequences"):
            ops.accept_tree(ids, ids, ids.int(), empty(2**24 + 1, dtype=I32), 1)
        with pytest.raises(ValueError, match="accept_tree: counts has too many sequences"):
            n = 2**18
            ops.accept_tree(ids, ids, ids.int(), empty(n + 1, dtype=I32), 1, empty(2, 64, 2, 64, 16, 64, dtype=BF16),
                            empty(n, 4, dtype=I32), empty(n, dtype=I32))  # fmt: skip
        pairs = empty(128, dtype=I32)
        with pytest.raises(ValueError, match="copy_blocks: src_blocks has too many blocks of this size"):
            ops.copy_blocks(empty(300, 16, 2, 64, 1024, 128), pairs, pairs)


def test_sample_tokens_without_settings_for_its_rows():
    # Without cu_seqlens_q every row has settings of its own: none at all are too few, not a call without work.
    assert sample_call(seqs=0) == INVALID and sample_call(seqs=0, rows=0) == OK and sample_call(seqs=0, cu=P) == OK
