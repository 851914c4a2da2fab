"""Performance cases of the tree, sampling and page operators over a paged cache.

One serving step over trees of drafted tokens runs ``tree_layout`` once (positions and masks from the drafts' parents), then per
layer the cache append and ``paged_tree`` (attention of the drafted nodes over the cache and their own ancestors), then
``sample_tokens`` on every node's logits, and at its end ``accept_tree`` (the drafted path that stands, and its keys and values
moved behind the sequence's own). ``copy_blocks`` copies pages of the cache: forked sequences, compaction.

``listed()`` gives the cases, ``draw(rng)`` more of the same ranges; ``prepare`` makes what a program holds before the
call, ``run`` is one pass (plain torch operations, or the framework's kernels where ``own`` is true), ``work`` what the
pass cannot do without and ``exact`` its result in float64.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
LAYERS, LAYER = 2, 1  # layers of an attention case's pool, and the one that it runs
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
WORD = 64  # rows in a word of a mask


# ------------------------------------------------------------------------------------------- cases
def _layout(name, seqs, nodes_lo, nodes_hi, start_hi):
    """``seqs`` trees of nodes_lo..nodes_hi nodes behind up to start_hi cached tokens."""
    case = {"kind": "layout", "seqs": seqs, "nodes_lo": nodes_lo, "nodes_hi": nodes_hi, "start_lo": 1, "start_hi": start_hi}
    return case if name is None else {"name": name, **case}


def _tree(name, seqs, nodes_lo, nodes_hi, start_lo, start_hi, heads, kv_heads, dim, dtype, block_size=16):
    """``seqs`` trees of nodes_lo..nodes_hi nodes behind start_lo..start_hi cached tokens."""
    case = {"kind": "tree", "seqs": seqs, "nodes_lo": nodes_lo, "nodes_hi": nodes_hi, "start_lo": start_lo, "start_hi": start_hi,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "block_size": block_size}  # fmt: skip
    return case if name is None else {"name": name, **case}


def _sample(name, rows, vocab, dtype, users, head):
    """``rows`` rows of logits for the given mix of users' settings; ``head``: a few likely tokens above the rest, as a language
    model's logits have them, else normal ones."""
    case = {"kind": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "users": users, "head": head}
    return case if name is None else {"name": name, **case}


def _accept(name, seqs, nodes_lo, nodes_hi, start_lo, start_hi, layers, kv_heads, dim, dtype, block_size=16):
    """``seqs`` trees, their tokens sampled; the pool has ``layers`` layers."""
    case = {"kind": "accept", "seqs": seqs, "nodes_lo": nodes_lo, "nodes_hi": nodes_hi, "start_lo": start_lo, "start_hi": start_hi,
            "layers": layers, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "block_size": block_size}  # fmt: skip
    return case if name is None else {"name": name, **case}


def _copy(name, pairs, partial, layers, kv_heads, dim, dtype, block_size=16):
    """``pairs`` pages copied, the first ``partial`` of them only in part."""
    case = {"kind": "copy", "pairs": pairs, "partial": partial, "layers": layers, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "block_size": block_size}  # fmt: skip
    return case if name is None else {"name": name, **case}


# (temperature, top_k, top_p, min_p) of the users of a batch, row after row. 0, 0, 1, 0: off.
USERS = {
    "one": [(0.8, 50, 0.95, 0.0)],
    "plain": [(1.0, 0, 1.0, 0.0), (0.7, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0)],
    "nucleus": [(1.0, 0, 0.9, 0.0), (0.7, 0, 0.95, 0.0)],
    "mixed": [(0.7, 50, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (0.8, 0, 1.0, 0.05), (1.0, 0, 1.0, 0.0),
              (1.2, 200, 0.99, 0.01), (1.0, 1, 1.0, 0.0), (0.9, 1000, 1.0, 0.0)],
}  # fmt: skip


def listed():
    return [
        # One user's tree of drafts: launch and latency count.
        _layout("layout_1", 1, 26, 26, 4000),
        # A full batch of large ragged trees, masks of several words.
        _layout("layout_128", 128, 65, 256, 8000),
        # One user: 64 drafted nodes part-way through a long answer.
        _tree("tree_1", 1, 64, 64, 4000, 4000, 32, 8, 128, "bf16"),
        # Ragged small trees of 32 sequences over long contexts.
        _tree("tree_32", 32, 9, 33, 1001, 8007, 32, 4, 64, "fp16", block_size=32),
        # A batch of 64-node trees over ragged contexts.
        _tree("tree_64", 64, 64, 64, 511, 4094, 32, 8, 128, "bf16"),
        # One user's next token.
        _sample("sample_1", 1, 50257, "fp32", "one", True),
        # A small batch without truncation, some users greedy.
        _sample("sample_48", 48, 50257, "bf16", "plain", False),
        # A full batch of users with settings of their own, over a large vocabulary.
        _sample("sample_256", 256, 128000, "fp32", "mixed", True),
        # One user's tree, in a pool of 12 layers of 12 heads.
        _accept("accept_1", 1, 26, 26, 700, 700, 12, 12, 64, "fp16"),
        # A full batch of trees.
        _accept("accept_64", 64, 33, 64, 100, 400, 16, 8, 128, "bf16"),
        # A request forked into four: the partly filled last page goes to each.
        _copy("copy_4", 4, 4, 12, 12, 64, "fp32"),
        # Pages moved together.
        _copy("copy_128", 128, 0, 16, 8, 128, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["layout", "tree", "tree", "sample", "sample", "accept", "copy"])
    if kind == "layout":
        lo = _log_int(rng, 1, 256)
        return _layout(None, _log_int(rng, 1, 128), lo, rng.randint(lo, 256), _log_int(rng, 1, 30000))
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    block_size = rng.choice([8, 16, 16, 32, 64])
    if kind == "sample":
        vocab = _log_int(rng, 1000, 128000)
        rows = min(_log_int(rng, 1, 512), max(1, 256 * 128000 // vocab))
        return _sample(None, rows, vocab, rng.choice(["fp32", "bf16", "fp16"]), rng.choice(sorted(USERS)), rng.random() < 0.7)
    if kind == "tree":
        group = rng.choice([1, 2, 3, 4, 7, 8])
        lo = _log_int(rng, 1, 100)
        hi = rng.randint(lo, min(130, 2 * lo + 5))
        start_lo = _log_int(rng, 1, 8000) - 1
        start_hi = rng.randint(start_lo, 2 * start_lo + 100)
        seqs = _log_int(rng, 1, 64)
        while seqs > 1 and seqs * kv_heads * dim * (start_hi + hi) * max(32, group * hi) > 64 * 8 * 128 * 4158 * 256 // 2:
            seqs -= 1
        return _tree(None, seqs, lo, hi, start_lo, start_hi, kv_heads * group, kv_heads, dim, rng.choice(["bf16", "fp16"]),
                     block_size)  # fmt: skip
    layers = rng.choice([1, 2, 6, 12, 16])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if kind == "accept":
        lo = _log_int(rng, 1, 64)
        start_lo = _log_int(rng, 1, 2000)
        return _accept(None, _log_int(rng, 1, 64), lo, rng.randint(lo, 64), start_lo, rng.randint(start_lo, 2 * start_lo), layers,
                       kv_heads, dim, rng.choice(["bf16", "fp16"]), min(block_size, 32))  # fmt: skip
    page = layers * 2 * kv_heads * dim * block_size * BYTES[dtype]
    pairs = min(_log_int(rng, 1, 512), max(1, 128 * 2**20 // page))
    return _copy(None, pairs, rng.randint(0, pairs), layers, kv_heads, dim, dtype, block_size)


# ------------------------------------------------------------------------------------------ shapes
def _spread(n, lo, hi, salt):
    """n lengths spread evenly over lo..hi, in a fixed shuffled order."""
    got = [lo + int((hi - lo + 1) * (i + 0.5) / n) for i in range(n)]
    random.Random(salt).shuffle(got)
    return got


def _lengths(case):
    """(cached tokens, nodes) of each sequence of a tree case."""
    nodes = _spread(case["seqs"], case["nodes_lo"], case["nodes_hi"], 1)
    return _spread(case["seqs"], case["start_lo"], case["start_hi"], 2), nodes


def _cdiv(a, b):
    return -(-a // b)


def _sums(counts):
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    return cu


# ------------------------------------------------------------------------------------------ inputs
def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device=DEVICE, generator=gen) * scale).to(dtype)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _grown(nodes, rng):
    """Parents of a tree's nodes: the last known token, then drafts grown from likely nodes, early ones most."""
    return [-1] + [int(i * rng.random() ** 1.5) for i in range(1, nodes)]


def _trees(case, rng):
    start, nodes = _lengths(case)
    parents = [_grown(n, rng) for n in nodes]
    return start, nodes, parents


def _words(case):
    return _cdiv(max(_lengths(case)[1]), WORD)


def _masks(parents, words):
    """Of each node: a bit for itself and for each ancestor."""
    got = []
    for p in parents:
        bits = []
        for i, at in enumerate(p):
            bits.append((bits[at] if at >= 0 else 0) | 1 << i)
        for b in bits:
            row = [b >> WORD * w & (1 << WORD) - 1 for w in range(words)]
            got.append([x - (1 << WORD) if x >> WORD - 1 else x for x in row])
    return got


def _prepare_layout(case, gen, rng):
    start, nodes, parents = _trees(case, rng)
    return {"case": case, "parents": _ints(sum(parents, [])), "cu": _ints(_sums(nodes)), "start": _ints(start),
            "max_new": max(nodes)}  # fmt: skip


def _tables(start, nodes, block_size, gen, spare, shared=False):
    """(tables, blocks): pages of sequences that grew side by side; ``shared``: whole pages of cached tokens are those of a
    common prompt, the rest their own."""
    need = [_cdiv(s + n, block_size) for s, n in zip(start, nodes)]
    common = max(s // block_size for s in start) if shared else 0
    mine = [k - min(common, s // block_size) for k, s in zip(need, start)]
    blocks = common + sum(mine) + spare
    ids = torch.randperm(blocks, device=DEVICE, generator=gen).int()
    tables = torch.zeros(len(nodes), max(need), dtype=torch.int32, device=DEVICE)
    for b, at in enumerate(_sums(mine)[:-1]):
        k = need[b] - mine[b]
        tables[b, :k] = ids[:k]
        tables[b, k : need[b]] = ids[common + at : common + at + mine[b]]
    return tables, blocks


def _prepare_tree(case, gen, rng):
    h, hk, d, bs = (case[k] for k in ("heads", "kv_heads", "dim", "block_size"))
    dtype = DTYPES[case["dtype"]]
    start, nodes, parents = _trees(case, rng)
    tables, blocks = _tables(start, nodes, bs, gen, 7)
    rows = sum(nodes)
    qkv = _randn(gen, rows, (h + 2 * hk) * d, dtype=dtype, scale=1.5)
    return {
        "case": case,
        "pool": _randn(gen, blocks, LAYERS, 2, hk, bs, d, dtype=dtype),
        "q": qkv[:, : h * d].view(rows, h, d),
        "out": torch.empty(rows, h, d, dtype=dtype, device=DEVICE),
        "tables": tables,
        "cu": _ints(_sums(nodes)),
        "start": _ints(start),
        "masks": _ints(_masks(parents, _words(case)), torch.int64),
        "max_new": max(nodes),
        "max_context": max(s + n for s, n in zip(start, nodes)),
    }


def _prepare_sample(case, gen, rng):
    rows, vocab = case["rows"], case["vocab"]
    if case["head"]:
        x = _randn(gen, rows, vocab, scale=2.0)
        many = min(512, vocab)
        rank = torch.arange(many, device=DEVICE, dtype=torch.float32)
        likely = 18.0 - (1.0 + torch.rand(rows, 1, device=DEVICE, generator=gen)) * torch.log1p(rank)[None, :]
        likely += 0.5 * _randn(gen, rows, many)
        at = torch.randperm(vocab, device=DEVICE, generator=gen)[:many]
        x[:, at] = likely[:, torch.randperm(many, device=DEVICE, generator=gen)]
    else:
        x = _randn(gen, rows, vocab, scale=3.0)
    users = [USERS[case["users"]][r % len(USERS[case["users"]])] for r in range(rows)]
    columns = [list(c) for c in zip(*users)]
    return {
        "case": case,
        "logits": x.to(DTYPES[case["dtype"]]),
        "uniforms": torch.rand(rows, device=DEVICE, generator=gen),
        "temperature": _ints(columns[0], torch.float32),
        "top_k": _ints(columns[1]),
        "top_p": _ints(columns[2], torch.float32),
        "min_p": _ints(columns[3], torch.float32),
    }


def _prepare_accept(case, gen, rng):
    hk, d, bs = case["kv_heads"], case["dim"], case["block_size"]
    start, nodes, parents = _trees(case, rng)
    tables, blocks = _tables(start, nodes, bs, gen, 3, shared=True)
    drafts, sampled = [], []
    for p in parents:
        mine = [rng.randrange(50257) for _ in p]
        children = [[] for _ in p]
        for i, at in enumerate(p):
            if at >= 0:
                children[at].append(i)
        # The target agrees with one of the drafts most of the time.
        sampled += [mine[rng.choice(c)] if c and rng.random() < 0.8 else rng.randrange(50257) for c in children]
        drafts += mine
    return {
        "case": case,
        "pool": _randn(gen, blocks, case["layers"], 2, hk, bs, d, dtype=DTYPES[case["dtype"]]),
        "tables": tables,
        "parents": _ints(sum(parents, [])),
        "drafts": _ints(drafts, torch.int64),
        "sampled": _ints(sampled, torch.int64),
        "cu": _ints(_sums(nodes)),
        "start": _ints(start),
        "max_new": max(nodes),
    }


def _prepare_copy(case, gen, rng):
    pairs, bs = case["pairs"], case["block_size"]
    blocks = 2 * pairs + 3
    ids = torch.randperm(blocks, device=DEVICE, generator=gen).int()
    slots = [rng.randint(1, bs) if i < case["partial"] else bs for i in range(pairs)]
    return {
        "case": case,
        "pool": _randn(gen, blocks, case["layers"], 2, case["kv_heads"], bs, case["dim"], dtype=DTYPES[case["dtype"]]),
        "src": ids[:pairs].clone(),
        "dst": ids[pairs : 2 * pairs].clone(),
        "slots": _ints(slots),
    }


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = random.Random(seed)
    make = {"layout": _prepare_layout, "tree": _prepare_tree, "sample": _prepare_sample, "accept": _prepare_accept,
            "copy": _prepare_copy}[case["kind"]]  # fmt: skip
    return make(case, gen, rng)


# ------------------------------------------------------------------------------------ plain forms
def _places(cu, max_new, fill):
    """(at, real) [seqs, max_new]: each sequence's rows, and which of them there are."""
    row = torch.arange(max_new, device=cu.device)
    real = row[None, :] < (cu[1:] - cu[:-1])[:, None]
    return torch.where(real, cu[:-1, None] + row[None, :], fill), real


def _plain_layout(s):
    cu, n = s["cu"].long(), s["max_new"]
    at, real = _places(cu, n, 0)
    parent = torch.where(real, s["parents"][at].long(), -1)
    row = torch.arange(n, device=cu.device)
    # Who leads to whom, in powers of two steps.
    seen = ((row[None, None, :] == parent[:, :, None]) | (row[None, :, None] == row[None, None, :])).float()
    for _ in range(max(1, (n - 1).bit_length())):
        seen = (torch.matmul(seen, seen.contiguous()) > 0).float()
    positions = s["start"].long()[:, None] + seen.sum(-1).long() - 1
    words = _cdiv(n, WORD)
    bits = torch.nn.functional.pad(seen.long(), (0, words * WORD - n)).view(-1, n, words, WORD)
    masks = (bits << torch.arange(WORD, device=cu.device)).sum(-1)
    return {"positions": positions[real], "masks": masks[real]}


def _plain_tree(s):
    case, q = s["case"], s["q"]
    hk, d, seqs = case["kv_heads"], case["dim"], case["seqs"]
    group, new, keys = case["heads"] // hk, s["max_new"], s["tables"].size(1) * case["block_size"]
    # [2, seqs, kv head, key, dim], padded to the longest table.
    kv = s["pool"][s["tables"].long(), LAYER].permute(2, 0, 3, 1, 4, 5).reshape(2, seqs, hk, keys, d)
    cu, start = s["cu"].long(), s["start"].long()
    at, real = _places(cu, new, 0)
    qp = q[at].float().view(seqs, new, hk, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, hk, group * new, d)
    scores = torch.matmul(qp, kv[0].float().transpose(-1, -2).contiguous()) / math.sqrt(d)
    bits = (s["masks"][at][..., None] >> torch.arange(WORD, device=q.device) & 1).bool().flatten(-2)  # [seqs, new, words * WORD]
    node = torch.arange(keys, device=q.device)[None, :] - start[:, None]  # [seqs, keys]
    inside = (node >= 0) & (node < bits.size(-1))
    marked = bits.gather(-1, torch.where(inside, node, 0)[:, None, :].expand(-1, new, -1)) & inside[:, None, :]
    seen = (node < 0)[:, None, :] | marked
    scores = scores.view(seqs, hk, group, new, keys).masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    weights = scores.exp_()
    total = weights.sum(-1, keepdim=True)
    # Slots behind a sequence's last key hold anything: no weight may meet them.
    values = kv[1].float().masked_fill_((node >= (cu[1:] - cu[:-1])[:, None])[:, None, :, None], 0.0)
    out = torch.matmul(weights.view(seqs, hk, group * new, keys), values).view(seqs, hk, group, new, d) / total
    return out.permute(0, 3, 1, 2, 4).reshape(seqs, new, hk * group, d)[real].to(q.dtype)


def _plain_sample(s):
    logits, t = s["logits"], s["temperature"][:, None].double()
    vocab = logits.size(1)
    x, order = torch.sort(logits.float(), dim=-1, descending=True, stable=True)
    x = x.double() / torch.where(t > 0, t, 1.0)
    w = (x - x[:, :1]).exp_()
    k = s["top_k"][:, None]
    w = torch.where((k <= 0) | (torch.arange(vocab, device=x.device)[None, :] < k), w, 0.0)
    before = w.cumsum(-1) - w
    p = s["top_p"][:, None].double()
    keep = (p >= 1) | (before < p * w.sum(-1, keepdim=True))
    keep &= w >= s["min_p"][:, None].double()
    keep[:, 0] = True
    w = torch.where(keep, w, 0.0)
    cum = torch.zeros_like(w).scatter_(1, order, w)
    last = vocab - 1 - (cum > 0).long().flip(-1).argmax(-1)
    cum = cum.cumsum(-1)
    token = torch.minimum((cum <= s["uniforms"][:, None].double() * cum[:, -1:]).sum(-1), last)
    return torch.where(t[:, 0] > 0, token, order[:, 0])


def _plain_accept(s):
    case, cu, start, pool = s["case"], s["cu"].long(), s["start"].long(), s["pool"]
    n, bs = s["max_new"], case["block_size"]
    at, real = _places(cu, n, 0)
    parent, draft, sampled = torch.where(real, s["parents"][at], -2), s["drafts"][at], s["sampled"][at]
    seqs = torch.arange(cu.numel() - 1, device=cu.device)
    tokens = torch.full((seqs.numel(), n), -1, dtype=torch.int64, device=cu.device)
    path = torch.full((seqs.numel(), n), -1, dtype=torch.int32, device=cu.device)
    node = torch.zeros_like(seqs)
    going = torch.ones_like(seqs, dtype=torch.bool)
    counts = torch.zeros_like(seqs)
    for step in range(min(n, 24)):  # (no listed or drawn tree is deeper)
        token = sampled[seqs, node]
        tokens[:, step] = torch.where(going, token, -1)
        path[:, step] = torch.where(going, node, -1).int()
        counts += going
        match = (parent == node[:, None]) & (draft == token[:, None])
        going &= match.any(-1)
        node = torch.where(going, match.long().argmax(-1), node)
    step = torch.arange(n, device=cu.device)
    b, j = torch.nonzero(step[None, :] < counts[:, None], as_tuple=True)
    src, dst = start[b] + path[b, j], start[b] + j
    moved = pool[s["tables"][b, src // bs].long(), :, :, :, src % bs]
    pool[s["tables"][b, dst // bs].long(), :, :, :, dst % bs] = moved
    return {"tokens": tokens, "path": path, "counts": counts.int(), "pool": pool}


def _plain_copy(s):
    pool, src, dst = s["pool"], s["src"].long(), s["dst"].long()
    filled = torch.arange(s["case"]["block_size"], device=pool.device)[None, :] < s["slots"][:, None]
    pool[dst] = torch.where(filled[:, None, None, None, :, None], pool[src], pool[dst])
    return pool


# ------------------------------------------------------------------------------------------- calls
def _own_layout(s):
    from tokquay_amd import ops

    positions, masks = ops.tree_layout(s["parents"], s["cu"], s["start"], s["max_new"])
    return {"positions": positions, "masks": masks}


def _own_tree(s):
    from tokquay_amd import ops

    ops.paged_tree(s["out"], s["q"], s["pool"], LAYER, s["tables"], s["cu"], s["start"], s["masks"], s["max_new"],
                   s["max_context"])  # fmt: skip
    return s["out"]


def _own_sample(s):
    from tokquay_amd import ops

    return ops.sample_tokens(s["logits"], s["uniforms"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])


def _own_accept(s):
    from tokquay_amd import ops

    tokens, path, counts = ops.accept_tree(s["sampled"], s["drafts"], s["parents"], s["cu"], s["max_new"], pool=s["pool"],
                                           block_tables=s["tables"], q_start=s["start"])  # fmt: skip
    return {"tokens": tokens, "path": path, "counts": counts, "pool": s["pool"]}


def _own_copy(s):
    from tokquay_amd import ops

    ops.copy_blocks(s["pool"], s["src"], s["dst"], s["slots"])
    return s["pool"]


@torch.no_grad()
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"layout": _own_layout, "tree": _own_tree, "sample": _own_sample, "accept": _own_accept, "copy": _own_copy}[kind](state)
    return {"layout": _plain_layout, "tree": _plain_tree, "sample": _plain_sample, "accept": _plain_accept,
            "copy": _plain_copy}[kind](state)  # fmt: skip


# -------------------------------------------------------------------------------------------- work
def work(case):
    """Each input read once, each output written once."""
    kind = case["kind"]
    if kind == "sample":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": rows * (vocab * BYTES[case["dtype"]] + 28), "flops": 4 * rows * vocab}
    if kind == "copy":
        bs = case["block_size"]
        slot = case["layers"] * 2 * case["kv_heads"] * case["dim"] * BYTES[case["dtype"]]
        slots = case["pairs"] * bs - case["partial"] * (bs - 1) / 2
        return {"bytes": 2 * slots * slot + 12 * case["pairs"], "flops": 0}
    start, nodes = _lengths(case)
    rows, seqs = sum(nodes), case["seqs"]
    if kind == "layout":
        return {"bytes": rows * (4 + 8 + 8 * _words(case)) + 8 * seqs, "flops": rows}
    if kind == "accept":
        # A few drafts of each tree stand and move.
        slot = case["layers"] * 2 * case["kv_heads"] * case["dim"] * BYTES[case["dtype"]]
        moved = sum(min(2, n - 1) for n in nodes)
        return {"bytes": rows * 20 + seqs * (12 * max(nodes) + 12) + 2 * slot * moved, "flops": 0}
    size = BYTES[case["dtype"]]
    visible = sum(s * n + n for s, n in zip(start, nodes))  # a node's ancestors among the drafts are few
    tables = 4 * sum(_cdiv(s + n, case["block_size"]) for s, n in zip(start, nodes))
    kv = 2 * sum(s + n for s, n in zip(start, nodes)) * case["kv_heads"] * case["dim"]
    return {"bytes": size * (kv + 2 * rows * case["heads"] * case["dim"]) + tables + rows * 8 * _words(case) + 12 * seqs,
            "flops": 4 * case["heads"] * case["dim"] * visible}  # fmt: skip


# ----------------------------------------------------------------------------------------- float64
def _ancestors(parents, i):
    """Node i and those above it, i first."""
    line = []
    while i >= 0:
        line.append(i)
        i = parents[i]
    return line


def _exact_layout(case, s):
    cu, parents, start = s["cu"].tolist(), s["parents"].tolist(), s["start"].tolist()
    positions, masks = [], []
    for b in range(case["seqs"]):
        mine = parents[cu[b] : cu[b + 1]]
        for i in range(len(mine)):
            line = _ancestors(mine, i)
            positions.append(start[b] + len(line) - 1)
            words = [0] * _words(case)
            for a in line:
                words[a // WORD] += 1 << a % WORD
            masks.append([w - (1 << WORD) if w >= 1 << WORD - 1 else w for w in words])
    return {"positions": torch.tensor(positions), "masks": torch.tensor(masks)}


def _exact_tree(case, s):
    start, nodes = _lengths(case)
    hk, bs = case["kv_heads"], case["block_size"]
    group = case["heads"] // hk
    words, q, out, at = s["masks"].tolist(), s["q"].double(), [], 0
    for b, (c, n) in enumerate(zip(start, nodes)):
        pos = torch.arange(c + n, device=DEVICE)
        slot = s["tables"][b].long()[pos // bs], pos % bs
        seen = [[words[at + i][j // WORD] >> j % WORD & 1 for j in range(n)] for i in range(n)]
        mask = torch.nn.functional.pad(torch.tensor(seen, device=DEVICE).bool(), (c, 0), value=True)
        rows = torch.empty(n, case["heads"], case["dim"], dtype=torch.float64, device=DEVICE)
        for h in range(hk):
            k, v = s["pool"][slot[0], LAYER, 0, h, slot[1]].double(), s["pool"][slot[0], LAYER, 1, h, slot[1]].double()
            for g in range(h * group, (h + 1) * group):
                x = (q[at : at + n, g] @ k.t()) * case["dim"] ** -0.5
                rows[:, g] = torch.softmax(torch.where(mask, x, -math.inf), dim=-1) @ v
        out.append(rows)
        at += n
    return torch.cat(out)


def _exact_sample(case, s):
    tokens = []
    settings = list(zip(*(s[k].tolist() for k in ("temperature", "top_k", "top_p", "min_p", "uniforms"))))
    for r, (t, k, p, low, u) in enumerate(settings):
        x = s["logits"][r].double()
        if t == 0:
            tokens.append(int(torch.argmax(x)))
            continue
        w = torch.exp((x - x.max()) / t)
        kept = torch.ones_like(w, dtype=torch.bool)
        if 0 < k < case["vocab"]:
            edge = float(torch.topk(x, k).values[-1])
            kept = x > edge
            ties = torch.nonzero(x == edge)[:, 0]
            kept[ties[: k - int(kept.sum())]] = True
        if p < 1:
            at = torch.nonzero(kept)[:, 0]
            at = at[torch.sort(x[at], descending=True, stable=True).indices]
            mass = torch.cumsum(w[at], 0)
            # The shortest beginning that reaches p of it.
            many = 1 + int(torch.searchsorted(mass, p * mass[-1:]))
            kept = torch.zeros_like(kept).index_fill_(0, at[:many], True)
        kept &= (w >= low) | (w == 1)
        at = torch.nonzero(kept)[:, 0]
        edges = torch.cumsum(w[at], 0)
        j = int(torch.searchsorted(edges, u * edges[-1:], right=True))
        tokens.append(int(at[min(j, at.numel() - 1)]))
    return torch.tensor(tokens)


def _exact_accept(case, s):
    cu, parents, drafts, sampled = (s[k].tolist() for k in ("cu", "parents", "drafts", "sampled"))
    tables, start, bs = s["tables"].tolist(), s["start"].tolist(), case["block_size"]
    shape = (case["seqs"], s["max_new"])
    tokens, path = torch.full(shape, -1, dtype=torch.int64), torch.full(shape, -1, dtype=torch.int32)
    counts, old = torch.zeros(case["seqs"], dtype=torch.int32), s["pool"]
    pool = old.double()
    for b in range(case["seqs"]):
        lo, n = cu[b], cu[b + 1] - cu[b]
        node = 0
        while node is not None:
            j = int(counts[b])
            path[b, j], tokens[b, j] = node, sampled[lo + node]
            src, dst = start[b] + node, start[b] + j
            pool[tables[b][dst // bs], :, :, :, dst % bs] = old[tables[b][src // bs], :, :, :, src % bs].double()
            counts[b] = j + 1
            node = next((i for i in range(n) if parents[lo + i] == node and drafts[lo + i] == sampled[lo + node]), None)
    return {"tokens": tokens, "path": path, "counts": counts, "pool": pool}


def _exact_copy(case, s):
    pool = s["pool"].double()
    for a, b, n in zip(s["src"].tolist(), s["dst"].tolist(), s["slots"].tolist()):
        pool[b, ..., :n, :] = s["pool"][a, ..., :n, :].double()
    return pool


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    return {"layout": _exact_layout, "tree": _exact_tree, "sample": _exact_sample, "accept": _exact_accept,
            "copy": _exact_copy}[case["kind"]](case, state)  # fmt: skip
