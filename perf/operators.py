"""Performance cases of the drafted-token and chunk operators over a 16-bit paged cache.

One serving step of new tokens (prompt chunks, drafted tokens, single tokens) runs, per layer, ``rope_cache_write``
(queries and keys normed and rotated, keys and values appended to the pool) and ``paged_chunk`` (attention of the new
rows over the pool), and at its end ``verify_drafts`` (drafted tokens against the target's logits).

``listed()`` gives the cases, ``draw(rng)`` more of the same ranges; ``prepare`` makes what a program holds before the
call, ``run`` is one pass (plain torch operations, or the framework's kernels where ``own`` is true), ``work`` what the
pass cannot do without and ``exact`` its result in float64.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
LAYERS, LAYER = 2, 1  # layers of the pool, and the one that a case runs
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


# ------------------------------------------------------------------------------------------- cases
def _rope(name, tokens, heads, kv_heads, dim, dtype, rotary, interleaved=False, norm=False, padded=0, block_size=16):
    """``tokens`` rows, ``padded`` of them without a slot; ``rotary`` of ``dim`` dims rotated."""
    case = {"kind": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "rotary": rotary, "interleaved": interleaved, "norm": norm, "padded": padded, "block_size": block_size}  # fmt: skip
    return case if name is None else {"name": name, **case}


def _chunk(name, seqs, new_lo, new_hi, start_lo, start_hi, heads, kv_heads, dim, dtype, block_size=16):
    """``seqs`` sequences feeding new_lo..new_hi tokens behind start_lo..start_hi cached ones."""
    case = {"kind": "chunk", "seqs": seqs, "new_lo": new_lo, "new_hi": new_hi, "start_lo": start_lo, "start_hi": start_hi,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "block_size": block_size}  # fmt: skip
    return case if name is None else {"name": name, **case}


def _verify(name, seqs, draft_lo, draft_hi, vocab, dtype, probs, greedy=0.0):
    """``seqs`` sequences of draft_lo..draft_hi drafted tokens; ``greedy``: the share of them at temperature 0."""
    case = {"kind": "verify", "seqs": seqs, "draft_lo": draft_lo, "draft_hi": draft_hi, "vocab": vocab, "dtype": dtype,
            "probs": probs, "greedy": greedy}  # fmt: skip
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # One user's next token: launch and latency count.
        _rope("rope_append_1", 1, 32, 8, 128, "bf16", 128),
        # A step's prompt chunks at a large token budget, queries and keys normed for each head.
        _rope("rope_append_8192", 8192, 32, 8, 128, "bf16", 128, norm=True),
        # A padded ragged step of a model that rotates half of each head in neighbouring pairs.
        _rope("rope_append_777", 777, 16, 16, 64, "fp16", 32, interleaved=True, padded=77, block_size=32),
        # One user, one token, part-way through a long answer.
        _chunk("chunk_token_1", 1, 1, 1, 4000, 4000, 32, 8, 128, "bf16"),
        # A full decode batch of ragged contexts: one token each.
        _chunk("chunk_tokens_128", 128, 1, 1, 511, 4094, 32, 8, 128, "bf16"),
        # Verification: the last token and a few drafted ones of 32 sequences over long contexts.
        _chunk("chunk_drafts_32", 32, 4, 6, 1001, 8007, 32, 4, 64, "fp16", block_size=32),
        # Chunked prefill of long prompts: 2,048 tokens each behind up to 6,144 cached ones.
        _chunk("chunk_prefill_4", 4, 2048, 2048, 0, 6144, 32, 8, 128, "bf16"),
        # The last ragged piece of one very long prompt.
        _chunk("chunk_piece_1", 1, 259, 259, 32500, 32500, 32, 8, 128, "bf16", block_size=64),
        # Whole ragged prompts admitted in one step, as many K/V heads as query heads, block size 16.
        _chunk("chunk_prompts_16", 16, 17, 1023, 0, 0, 12, 12, 64, "fp16"),
        # One user's four drafted tokens.
        _verify("verify_1", 1, 4, 4, 50257, "fp32", True),
        # A batch of ragged drafts from looking the prompt up (no draft probabilities), some users greedy.
        _verify("verify_64", 64, 0, 7, 50257, "bf16", False, greedy=0.25),
        # A full batch with a draft model's probabilities over a large vocabulary.
        _verify("verify_128", 128, 4, 4, 128000, "fp32", True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "chunk", "chunk", "verify"])
    if kind == "rope":
        dim = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 4, 8, 12])
        tokens = _log_int(rng, 1, 8192)
        interleaved = rng.random() < 0.3
        return _rope(None, tokens, kv_heads * rng.choice([1, 2, 3]), kv_heads, dim, rng.choice(["bf16", "fp16", "fp32"]),
                     rng.choice([dim, dim, dim // 2, dim // 4]), interleaved, rng.random() < 0.5,
                     rng.choice([0, tokens // 9]), rng.choice([8, 16, 32, 64]))  # fmt: skip
    if kind == "verify":
        vocab = _log_int(rng, 1000, 128000)
        lo = rng.randint(0, 7)
        hi = rng.randint(lo, 8)
        seqs = min(_log_int(rng, 1, 256), max(1, 640 * 128000 // (vocab * (hi + 1))))
        return _verify(None, seqs, lo, hi, vocab, rng.choice(["fp32", "bf16", "fp16"]), rng.random() < 0.5,
                       rng.choice([0.0, 0.3]))  # fmt: skip
    dim = rng.choice([64, 128])
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8])
    form = rng.choice(["token", "drafts", "chunk"])
    new_lo = {"token": 1, "drafts": rng.randint(2, 5), "chunk": _log_int(rng, 17, 2048)}[form]
    new_hi = {"token": 1, "drafts": rng.randint(5, 9), "chunk": rng.randint(new_lo, min(2048, 2 * new_lo))}[form]
    start_lo = _log_int(rng, 1, 8000) - 1
    start_hi = rng.randint(start_lo, min(32768, 2 * start_lo + 100))
    seqs = _log_int(rng, 1, 16 if form == "chunk" else 128)
    while seqs > 1 and (seqs * kv_heads * group * new_hi * (start_hi + new_hi) * dim > 4 * 32 * 2048 * 8192 * 128 * 0.6
                        or seqs * kv_heads * group * new_hi * (start_hi + new_hi) > 4 * 32 * 2048 * 8192
                        or seqs * kv_heads * dim * (start_hi + new_hi) > 128 * 8 * 128 * 4095):  # fmt: skip
        seqs -= 1
    return _chunk(None, seqs, new_lo, new_hi, start_lo, start_hi, kv_heads * group, kv_heads, dim,
                  rng.choice(["bf16", "fp16"]), rng.choice([8, 16, 16, 32, 64]))  # fmt: skip


# ------------------------------------------------------------------------------------------ shapes
def _spread(n, lo, hi, salt):
    """n lengths spread evenly over lo..hi, in a fixed shuffled order."""
    got = [lo + int((hi - lo + 1) * (i + 0.5) / n) for i in range(n)]
    random.Random(salt).shuffle(got)
    return got


def _lengths(case):
    """(cached, fed) token counts of each sequence of a chunk case."""
    new = _spread(case["seqs"], case["new_lo"], case["new_hi"], 1)
    return _spread(case["seqs"], case["start_lo"], case["start_hi"], 2), new


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


def _prepare_rope(case, gen, rng):
    n, h, hk, d, bs = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "block_size"))
    dtype = DTYPES[case["dtype"]]
    blocks = _cdiv(n, bs) + 5
    qkv = _randn(gen, n, (h + 2 * hk) * d, dtype=dtype)  # rows are views of the fused projection's output
    token = torch.arange(n, device=DEVICE)  # a prompt's tokens, in blocks taken from all over the pool
    slots = torch.randperm(blocks, device=DEVICE, generator=gen)[token // bs] * bs + token % bs
    if case["padded"]:
        slots[torch.randperm(n, device=DEVICE, generator=gen)[: case["padded"]]] = -1
    max_pos = 16384
    r = case["rotary"]
    angles = torch.arange(max_pos, dtype=torch.float64, device=DEVICE)[:, None] * _frequencies(r)[None, :]
    state = {
        "case": case,
        "pool": _randn(gen, blocks, LAYERS, 2, hk, bs, d, dtype=dtype),
        "qkv": qkv,
        "q": qkv[:, : h * d].view(n, h, d),
        "k": qkv[:, h * d : (h + hk) * d].view(n, hk, d),
        "v": qkv[:, (h + hk) * d :].view(n, hk, d),
        "q_out": torch.empty(n, h, d, dtype=dtype, device=DEVICE),
        "slots": slots,
        "positions": torch.randint(0, max_pos, (n,), device=DEVICE, generator=gen),
        "table": torch.cat([angles.cos(), angles.sin()], dim=1).float(),
        "q_norm": None,
        "k_norm": None,
    }
    if case["norm"]:
        state["q_norm"] = (1 + 0.2 * _randn(gen, d)).to(dtype)
        state["k_norm"] = (1 + 0.2 * _randn(gen, d)).to(dtype)
    return state


def _frequencies(rotary):
    half = rotary // 2
    return 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / half)


def _prepare_chunk(case, gen, rng):
    h, hk, d, bs = (case[k] for k in ("heads", "kv_heads", "dim", "block_size"))
    dtype = DTYPES[case["dtype"]]
    start, new = _lengths(case)
    need = [_cdiv(s + n, bs) for s, n in zip(start, new)]
    blocks = sum(need) + 7
    ids = torch.randperm(blocks, device=DEVICE, generator=gen).int()  # sequences that grew side by side
    tables = torch.zeros(len(new), max(need), dtype=torch.int32, device=DEVICE)
    for b, (at, k) in enumerate(zip(_sums(need), need)):
        tables[b, :k] = ids[at : at + k]
    rows = sum(new)
    qkv = _randn(gen, rows, (h + 2 * hk) * d, dtype=dtype, scale=1.5)
    return {
        "case": case,
        "pool": _randn(gen, blocks, LAYERS, 2, hk, bs, d, dtype=dtype),
        "q": qkv[:, : h * d].view(rows, h, d),
        "out": torch.empty(rows, h, d, dtype=dtype, device=DEVICE),
        "tables": tables,
        "cu": _ints(_sums(new)),
        "start": _ints(start),
        "max_new": max(new),
        "max_context": max(s + n for s, n in zip(start, new)),
    }


def _prepare_verify(case, gen, rng):
    seqs, vocab = case["seqs"], case["vocab"]
    drafts = _spread(seqs, case["draft_lo"], case["draft_hi"], 3)
    cu = _sums([n + 1 for n in drafts])
    rows = cu[-1]
    owner = torch.repeat_interleave(torch.arange(seqs, device=DEVICE), _ints([n + 1 for n in drafts], torch.int64))
    temps = [0.0 if rng.random() < case["greedy"] else rng.choice([0.6, 0.8, 1.0]) for _ in range(seqs)]
    temperature = torch.tensor(temps, device=DEVICE)
    # Peaked target logits; the draft model's are near them, and drafts are drawn from it.
    logits = _randn(gen, rows, vocab, dtype=DTYPES[case["dtype"]], scale=3.0)
    near = logits.float() + _randn(gen, rows, vocab, scale=0.5)
    state = {"case": case, "logits": logits, "cu": _ints(cu), "temperature": temperature, "max_rows": max(drafts) + 1,
             "uniforms": torch.rand(rows, device=DEVICE, generator=gen), "probs": None}  # fmt: skip
    if case["probs"]:
        t = temperature[owner][:, None]
        soft = torch.softmax(near / torch.where(t > 0, t, 1.0), dim=-1)
        hard = torch.nn.functional.one_hot(near.argmax(-1), vocab).float()
        state["probs"] = torch.where(t > 0, soft, hard)
        state["drafts"] = torch.multinomial(state["probs"], 1, generator=gen)[:, 0]
    else:
        state["drafts"] = near.argmax(-1)
    return state


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = random.Random(seed)
    make = {"rope": _prepare_rope, "chunk": _prepare_chunk, "verify": _prepare_verify}[case["kind"]]
    return make(case, gen, rng)


# ------------------------------------------------------------------------------------ plain forms
def _plain_norm(x, weight):
    if weight is None:
        return x
    return x / torch.sqrt(torch.mean(x * x, dim=-1, keepdim=True) + EPS) * weight.float()


def _plain_rotate(x, table, positions, interleaved):
    half = table.size(1) // 2
    at = table[positions][:, None, :]
    cos, sin = at[..., :half], at[..., half:]
    turned, rest = x[..., : 2 * half], x[..., 2 * half :]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _plain_rope(s):
    case, pool = s["case"], s["pool"]
    turn = lambda x, w: _plain_rotate(_plain_norm(x.float(), w), s["table"], s["positions"], case["interleaved"])  # noqa: E731
    q, k = turn(s["q"], s["q_norm"]).to(pool.dtype), turn(s["k"], s["k_norm"]).to(pool.dtype)
    kept = s["slots"] >= 0
    slots = s["slots"][kept]
    block, off = slots // case["block_size"], slots % case["block_size"]
    pool[block, LAYER, 0, :, off] = k[kept]
    pool[block, LAYER, 1, :, off] = s["v"][kept]
    return {"q": q, "pool": pool}


def _plain_chunk(s):
    case, q = s["case"], s["q"]
    hk, d, seqs = case["kv_heads"], case["dim"], case["seqs"]
    group, new, keys = case["heads"] // hk, s["max_new"], s["tables"].size(1) * case["block_size"]
    # [2, seqs, kv head, key, dim], padded to the longest table.
    kv = s["pool"][s["tables"].long(), LAYER].permute(2, 0, 3, 1, 4, 5).reshape(2, seqs, hk, keys, d)
    cu, start = s["cu"].long(), s["start"].long()
    row = torch.arange(new, device=q.device)
    real = row[None, :] < (cu[1:] - cu[:-1])[:, None]  # [seqs, new]
    at = torch.where(real, cu[:-1, None] + row[None, :], 0)
    qp = q[at].float().view(seqs, new, hk, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, hk, group * new, d)
    scores = torch.matmul(qp, kv[0].float().transpose(-1, -2).contiguous()) / math.sqrt(d)
    unseen = torch.arange(keys, device=q.device)[None, None, :] > (start[:, None] + row[None, :])[:, :, None]
    scores = scores.view(seqs, hk, group, new, keys).masked_fill_(unseen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    weights = scores.exp_()
    total = weights.sum(-1, keepdim=True)
    # Slots behind a sequence's last key hold anything: no weight may meet them.
    values = kv[1].float().masked_fill_(torch.arange(keys, device=q.device)[None, None, :, None]
                                        >= (start + cu[1:] - cu[:-1])[:, None, None, None], 0.0)  # fmt: skip
    out = torch.matmul(weights.view(seqs, hk, group * new, keys), values).view(seqs, hk, group, new, d) / total
    return out.permute(0, 3, 1, 2, 4).reshape(seqs, new, hk * group, d)[real].to(q.dtype)


def _plain_verify(s):
    logits, cu, probs, drafts = s["logits"], s["cu"].long(), s["probs"], s["drafts"]
    rows, vocab = logits.shape
    counts = cu[1:] - cu[:-1]
    owner = torch.repeat_interleave(torch.arange(counts.numel(), device=logits.device), counts, output_size=rows)
    t = s["temperature"][owner][:, None].double()
    x = logits.double() / torch.where(t > 0, t, 1.0)
    x -= x.amax(-1, keepdim=True)
    p = x.exp_()
    p /= p.sum(-1, keepdim=True)
    best = torch.zeros_like(p).scatter_(1, logits.argmax(-1, keepdim=True), 1.0)
    p = torch.where(t > 0, p, best)
    row = torch.arange(rows, device=logits.device)
    qx = torch.ones(rows, dtype=torch.float64, device=logits.device) if probs is None else probs[row, drafts].double()
    accept = s["uniforms"].double() * qx < p[row, drafts]
    step = torch.arange(s["max_rows"], device=logits.device)
    drafted = step[None, :] < (counts - 1)[:, None]
    at = torch.where(drafted, cu[:-1, None] + step[None, :], 0)
    accepted = (accept[at] & drafted).long().cumprod(-1).sum(-1)
    rejected = (accepted < counts - 1)[:, None]
    chosen = cu[:-1] + accepted
    ps = p[chosen]
    if probs is None:
        rest = ps.scatter(1, drafts[chosen][:, None], 0.0)
    else:
        rest = torch.clamp(ps - probs[chosen].double(), min=0.0)
    w = torch.where(rejected & (rest.sum(-1, keepdim=True) > 0), rest, ps)
    cum = w.cumsum(-1)
    goal = s["uniforms"][cu[1:] - 1].double()[:, None] * cum[:, -1:]
    token = torch.minimum((cum <= goal).sum(-1), vocab - 1 - (w > 0).long().flip(-1).argmax(-1))
    tokens = torch.where(step[None, :] < accepted[:, None], drafts[at], -1)
    tokens.scatter_(1, accepted[:, None], token[:, None])
    return {"tokens": tokens, "accepted": accepted.int()}


# ------------------------------------------------------------------------------------------- calls
def _own_rope(s):
    from tokquay_amd import ops

    ops.rope_cache_write(s["q_out"], s["q"], s["k"], s["v"], s["pool"], LAYER, s["slots"], s["positions"], s["table"],
                         interleaved=s["case"]["interleaved"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)  # fmt: skip
    return {"q": s["q_out"], "pool": s["pool"]}


def _own_chunk(s):
    from tokquay_amd import ops

    ops.paged_chunk(s["out"], s["q"], s["pool"], LAYER, s["tables"], s["cu"], s["start"], s["max_new"], s["max_context"])
    return s["out"]


def _own_verify(s):
    from tokquay_amd import ops

    tokens, accepted = ops.verify_drafts(s["logits"], s["drafts"], s["uniforms"], s["cu"], s["max_rows"],
                                         s["temperature"], draft_probs=s["probs"])  # fmt: skip
    return {"tokens": tokens, "accepted": accepted}


@torch.no_grad()
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rope": _own_rope, "chunk": _own_chunk, "verify": _own_verify}[kind](state)
    return {"rope": _plain_rope, "chunk": _plain_chunk, "verify": _plain_verify}[kind](state)


# -------------------------------------------------------------------------------------------- work
def work(case):
    """Each input read once, each output written once."""
    if case["kind"] == "rope":
        n, width = case["tokens"], (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        stored = n * case["heads"] * case["dim"] + 2 * (n - case["padded"]) * case["kv_heads"] * case["dim"]
        turned = n * (case["heads"] + case["kv_heads"])
        return {"bytes": BYTES[case["dtype"]] * (n * width + stored) + n * (4 * case["rotary"] + 16),
                "flops": turned * (3 * case["rotary"] + (4 * case["dim"] if case["norm"] else 0))}  # fmt: skip
    if case["kind"] == "chunk":
        start, new = _lengths(case)
        size = BYTES[case["dtype"]]
        visible = sum(s * n + n * (n + 1) // 2 for s, n in zip(start, new))
        tables = 4 * sum(_cdiv(s + n, case["block_size"]) for s, n in zip(start, new))
        kv = 2 * sum(s + n for s, n in zip(start, new)) * case["kv_heads"] * case["dim"]
        return {"bytes": size * (kv + 2 * sum(new) * case["heads"] * case["dim"]) + tables + 12 * len(new),
                "flops": 4 * case["heads"] * case["dim"] * visible}  # fmt: skip
    drafts = _spread(case["seqs"], case["draft_lo"], case["draft_hi"], 3)
    rows = sum(drafts) + len(drafts)
    # Of the draft's probabilities: each drafted token's, and one row for each sequence.
    probs = 4 * (sum(drafts) + case["seqs"] * case["vocab"]) if case["probs"] else 0
    return {"bytes": rows * case["vocab"] * BYTES[case["dtype"]] + probs + 20 * rows + 12 * case["seqs"],
            "flops": 4 * rows * case["vocab"]}  # fmt: skip


# ----------------------------------------------------------------------------------------- float64
def _exact_rope(case, s):
    n, r, bs = case["tokens"], case["rotary"], case["block_size"]
    angle = s["positions"].double()[:, None] * _frequencies(r)[None, :]  # [n, r / 2]
    first = torch.arange(r // 2, device=DEVICE) * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else r // 2)

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
        # A rotation in the complex plane.
        z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(angle), angle)[:, None, :]
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    pool = s["pool"].double()
    flat = pool[:, LAYER].permute(0, 3, 1, 2, 4).reshape(-1, 2, case["kv_heads"], case["dim"])  # by slot
    kept = s["slots"] >= 0
    flat[s["slots"][kept]] = torch.stack([turned(s["k"], s["k_norm"]), s["v"].double()], dim=1)[kept]
    pool[:, LAYER] = flat.view(-1, bs, 2, case["kv_heads"], case["dim"]).permute(0, 2, 3, 1, 4)
    return {"q": turned(s["q"], s["q_norm"]), "pool": pool}


def _exact_chunk(case, s):
    start, new = _lengths(case)
    hk, bs = case["kv_heads"], case["block_size"]
    group = case["heads"] // hk
    q, out, at = s["q"].double(), [], 0
    for b, (c, n) in enumerate(zip(start, new)):
        pos = torch.arange(c + n, device=DEVICE)
        slot = s["tables"][b].long()[pos // bs], pos % bs
        mask = pos[None, :] <= pos[c:][:, None]
        rows = torch.empty(n, case["heads"], case["dim"], dtype=torch.float64, device=DEVICE)
        for h in range(hk):
            k, v = s["pool"][slot[0], LAYER, 0, h, slot[1]].double(), s["pool"][slot[0], LAYER, 1, h, slot[1]].double()
            for g in range(h * group, (h + 1) * group):
                x = (q[at : at + n, g] @ k.t()) * case["dim"] ** -0.5
                rows[:, g] = torch.softmax(torch.where(mask, x, -math.inf), dim=-1) @ v
        out.append(rows)
        at += n
    return torch.cat(out)


def _exact_verify(case, s):
    tokens = torch.full((case["seqs"], s["max_rows"]), -1, dtype=torch.int64)
    accepted = torch.zeros(case["seqs"], dtype=torch.int32)
    cu, drafts, temps = s["cu"].tolist(), s["drafts"].tolist(), s["temperature"].tolist()
    u = s["uniforms"].double().tolist()

    def target(row, t):
        if t == 0:
            return torch.nn.functional.one_hot(torch.argmax(s["logits"][row]), case["vocab"]).double()
        return torch.softmax(s["logits"][row].double() / t, dim=-1)

    for b in range(case["seqs"]):
        lo, last = cu[b], cu[b + 1] - 1
        i = 0
        while True:
            p = target(lo + i, temps[b])
            if lo + i == last:
                break
            x = drafts[lo + i]
            q = torch.zeros_like(p).index_fill_(0, torch.tensor([x], device=DEVICE), 1.0)
            q = q if s["probs"] is None else s["probs"][lo + i].double()
            if u[lo + i] * float(q[x]) >= float(p[x]):
                more = (p - q).relu()
                p = more if float(more.sum()) > 0 else p
                break
            tokens[b, i] = x
            i += 1
        edges = torch.cumsum(p, 0)
        goal = u[last] * float(edges[-1])
        at = int(torch.searchsorted(edges, torch.tensor([goal], dtype=torch.float64, device=DEVICE), right=True))
        tokens[b, i] = min(at, int(torch.nonzero(p)[-1]))
        accepted[b] = i
    return {"tokens": tokens, "accepted": accepted}


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    return {"rope": _exact_rope, "chunk": _exact_chunk, "verify": _exact_verify}[case["kind"]](case, state)
