"""The operators of serving in 8-bit integers, as timed cases with their plain forms.

Kinds:
  append   this pass's K / V rows into an int8 paged cache with a scale for
           every block of tokens and KV head, the rotary embedding applied to
           q and k on the way (`rope_kv_write`). A block's scale grows with the
           rows appended to it, and the rows it held are re-expressed with it.
  attend   attention out of such a cache (`paged_attention`): decode steps of
           one query per sequence, packed passes of prompt chunks over a cached
           prefix, and chunks with decode rows beside them.
  product  `x w^T` with x quantised to 8 bits with a scale for each row (token)
           and w held in 8 bits with a scale for each output channel
           (`linear_int8`): the engine's projections.

Sizes are those of the package's own configurations and benchmark (32 query /
8 KV heads, head_dim 128 or 64, blocks of 16 slots, the projections of the
Llama-3-8B architecture), odd and ragged ones among them.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = torch.device("cuda")
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
ROPE_THETA = 500000.0
STEP = 1.0 / 127.0  # a scale is the largest magnitude over 127
LEAST = 2.0 ** -126  # and no less than the smallest normal float32


def listed():
    return [
        # A small model's decode step over four sequences, eager: launches count.
        {"name": "append_step_4", "kind": "append", "seqs": 4, "lo": 1, "hi": 1, "kv_heads": 8, "groups": 4, "dim": 64,
         "block": 16, "dtype": "bf16", "lens": 1},
        # A decode step of a well-filled server.
        {"name": "append_step_128", "kind": "append", "seqs": 128, "lo": 1, "hi": 1, "kv_heads": 8, "groups": 4,
         "dim": 128, "block": 16, "dtype": "bf16", "lens": 2},
        # Ragged prompt chunks, together near the engine's token budget.
        {"name": "append_packed", "kind": "append", "seqs": 7, "lo": 300, "hi": 1400, "kv_heads": 8, "groups": 4,
         "dim": 128, "block": 16, "dtype": "bf16", "lens": 3},
        # The smallest attention call: four short contexts of a small model.
        {"name": "decode_4", "kind": "attend", "seqs": 4, "rows": 4, "qlo": 1, "qhi": 1, "lo": 37, "hi": 1023,
         "kv_heads": 8, "groups": 4, "dim": 64, "block": 16, "dtype": "bf16", "lens": 4},
        # The benchmark's decode step: 64 sequences of 512 .. 8192 keys.
        {"name": "decode_64", "kind": "attend", "seqs": 64, "rows": 64, "qlo": 1, "qhi": 1, "lo": 512, "hi": 8192,
         "kv_heads": 8, "groups": 4, "dim": 128, "block": 16, "dtype": "bf16", "lens": 5},
        # Long contexts over few sequences, what a cache of half the bytes is for.
        {"name": "decode_long", "kind": "attend", "seqs": 4, "rows": 4, "qlo": 1, "qhi": 1, "lo": 32768, "hi": 131072,
         "kv_heads": 8, "groups": 4, "dim": 128, "block": 16, "dtype": "f16", "lens": 6},
        # A follow-up question: one short chunk over a cached conversation, small heads.
        {"name": "packed_small", "kind": "attend", "seqs": 1, "rows": 0, "qlo": 101, "qhi": 101, "lo": 4096, "hi": 4096,
         "kv_heads": 8, "groups": 4, "dim": 64, "block": 16, "dtype": "bf16", "lens": 7},
        # Continuous batching: ragged chunks beside decode rows.
        {"name": "packed_mixed", "kind": "attend", "seqs": 36, "rows": 28, "qlo": 64, "qhi": 1024, "lo": 0, "hi": 4096,
         "kv_heads": 8, "groups": 4, "dim": 128, "block": 16, "dtype": "bf16", "lens": 8},
        # Long prompts in chunks: 2048 queries over 8192 cached keys.
        {"name": "packed_long", "kind": "attend", "seqs": 3, "rows": 0, "qlo": 2048, "qhi": 2048, "lo": 8192, "hi": 8192,
         "kv_heads": 8, "groups": 4, "dim": 128, "block": 16, "dtype": "bf16", "lens": 9},
        # One user's decode step: the fused q / k / v projection of a single row.
        {"name": "product_1", "kind": "product", "rows": 1, "k": 4096, "n": 6144, "dtype": "bf16"},
        # A decode batch through the MLP's down projection.
        {"name": "product_61", "kind": "product", "rows": 61, "k": 14336, "n": 4096, "dtype": "f16"},
        # A prompt pass through the MLP's gate and up projection.
        {"name": "product_4099", "kind": "product", "rows": 4099, "k": 4096, "n": 28672, "dtype": "bf16"},
    ]


def draw(rng):
    """One more case: sizes spread over the ranges the listed cases stand for."""
    def spread(lo, hi):  # log-uniform whole number
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["append", "append", "attend", "attend", "attend", "product", "product"])
    dtype = "bf16" if rng.random() < 0.7 else "f16"
    if kind == "product":
        k, n = spread(64, 14336), spread(64, 28672)
        return {"kind": kind, "rows": spread(1, min(8192, 4099 * 4096 * 28672 // (k * n))), "k": k, "n": n, "dtype": dtype}
    kv_heads, groups = (8, 4) if rng.random() < 0.5 else (rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 5, 8, 16]))
    case = {"kind": kind, "kv_heads": kv_heads, "groups": groups, "dim": rng.choice([64, 128]),
            "block": rng.choice([16, 16, 16, 8, 32]), "dtype": dtype, "lens": rng.randrange(1 << 30)}
    if kind == "append":
        if rng.random() < 0.5:
            return case | {"seqs": spread(1, 256), "lo": 1, "hi": 1}
        seqs = rng.randint(1, 8)
        hi = spread(4, 8192 // seqs)
        return case | {"seqs": seqs, "lo": max(1, hi // 4), "hi": hi}
    if rng.random() < 0.5:  # a decode step; values of the cache held to those of the largest listed one
        hi = spread(64, 131072)
        most = 330000 * 8 * 128 // (kv_heads * case["dim"]) // hi
        seqs = spread(1, max(1, min(256, most)))
        return case | {"seqs": seqs, "rows": seqs, "qlo": 1, "qhi": 1, "lo": max(1, hi // 16), "hi": hi}
    qhi, hi = spread(8, 2048), spread(1, 8192)
    chunks = rng.randint(1, 6)
    while chunks > 1 and chunks * qhi * (hi + qhi) * kv_heads * groups * case["dim"] > 2.4e11:
        chunks -= 1
    while qhi > 8 and chunks * qhi * (hi + qhi) * kv_heads * groups * case["dim"] > 2.4e11:
        qhi //= 2
    rows = rng.choice([0, 0, spread(1, 32)])
    return case | {"seqs": chunks + rows, "rows": rows, "qlo": max(2, qhi // 8), "qhi": qhi, "lo": 0, "hi": hi}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _lengths(case):
    """(first position, tokens) of each sequence of an append, (queries, keys before them) of an attention pass."""
    rng = random.Random(case["lens"])
    if case["kind"] == "append":
        return [(rng.randint(0, 8191), rng.randint(case["lo"], case["hi"])) for _ in range(case["seqs"])]
    lens = [(rng.randint(case["qlo"], case["qhi"]), rng.randint(case["lo"], case["hi"]))
            for _ in range(case["seqs"] - case["rows"])]
    # A row's keys count its own.
    return lens + [(1, rng.randint(max(1, case["lo"]), max(1, case["hi"])) - 1) for _ in range(case["rows"])]


def _randn(shape, gen):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32)


def _cache(blocks, case, gen, spread):
    """An int8 store of random rows: codes [slots, heads, dim], scales [blocks, heads] whose magnitudes spread e^N(0, spread)."""
    shape = (blocks, case["block"], case["kv_heads"], case["dim"])
    codes = torch.empty(shape, dtype=torch.int8, device=DEVICE)
    scales = torch.empty(blocks, case["kv_heads"], device=DEVICE)
    per = max(1, (1 << 27) // (case["block"] * case["kv_heads"] * case["dim"]))
    for b in range(0, blocks, per):
        x = _randn((min(per, blocks - b), *shape[1:]), gen)
        s = x.abs().amax(dim=(1, 3)) * STEP
        codes[b:b + per] = torch.round(x / s[:, None, :, None]).to(torch.int8)
        scales[b:b + per] = s * torch.exp(spread * _randn(s.shape, gen))
    return codes.view(-1, *shape[2:]), scales


def _blocks_of(lens, block, gen):
    """Each sequence's blocks out of a shuffled run, for the positions [first, first + count) of `lens`, and how many there are."""
    counts = [(s + c - 1) // block - s // block + 1 for s, c in lens]
    order = torch.randperm(sum(counts), generator=gen, device=DEVICE)
    return order.split(counts), sum(counts)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "product":
        rows, k, n = case["rows"], case["k"], case["n"]
        x = _randn((rows, k), gen) * torch.exp(0.5 * _randn((rows, 1), gen))
        w = _randn((n, k), gen) * 0.02
        scale = w.abs().amax(dim=1) * STEP
        # Rows of codes start at multiples of 16 bytes, as `quantize_weight` lays them out.
        codes = torch.zeros(n, -(-k // 16) * 16, dtype=torch.int8, device=DEVICE)[:, :k]
        codes.copy_(torch.round(w / scale[:, None]))
        return {"case": case, "x": x.to(dtype), "codes": codes, "scale": scale}
    lens, block = _lengths(case), case["block"]
    heads, kv_heads, dim = case["kv_heads"] * case["groups"], case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        # The store holds the blocks written to: what an append reads and writes of a cache.
        tables, blocks = _blocks_of(lens, block, gen)
        keys, key_scales = _cache(blocks, case, gen, 0.5)
        values, value_scales = _cache(blocks, case, gen, 0.5)
        step = case["hi"] == 1
        positions = torch.cat([torch.arange(s, s + c, device=DEVICE) for s, c in lens])
        slots = torch.cat([t[torch.arange(s, s + c, device=DEVICE) // block - s // block] * block
                           + torch.arange(s, s + c, device=DEVICE) % block for t, (s, c) in zip(tables, lens)])
        inv_freq = ROPE_THETA ** (-torch.arange(0, dim, 2, device=DEVICE, dtype=torch.float64) / dim)
        angles = positions[:, None] * inv_freq
        angles = torch.cat((angles, angles), dim=1)
        tokens = positions.numel()
        lead = (tokens, 1) if step else (1, tokens)  # [batch, tokens] of a decode step, of a packed pass
        qkv = _randn((*lead, heads + 2 * kv_heads, dim), gen).to(dtype)
        q, k, v = (t.transpose(1, 2) for t in qkv.split((heads, kv_heads, kv_heads), dim=2))
        return {"case": case, "q": q, "k": k, "v": v, "slots": slots[None],
                "cos": angles.cos().to(dtype).view(*lead, dim), "sin": angles.sin().to(dtype).view(*lead, dim),
                "keys": keys, "values": values, "key_scales": key_scales, "value_scales": value_scales}
    contexts = [q + p for q, p in lens]
    tables, blocks = _blocks_of([(0, c) for c in contexts], block, gen)
    keys, key_scales = _cache(blocks, case, gen, 0.2)
    values, value_scales = _cache(blocks, case, gen, 0.5)
    width = max(contexts)
    at = torch.arange(width, device=DEVICE)
    table = torch.zeros(len(lens), width, dtype=torch.int64, device=DEVICE)
    for i, t in enumerate(tables):
        table[i, :contexts[i]] = t[at[:contexts[i]] // block] * block + at[:contexts[i]] % block
    queries = [q for q, _ in lens]
    step = case["rows"] == case["seqs"]
    query = _randn((sum(queries), heads, dim), gen).to(dtype)
    starts = [0]
    for q in queries:
        starts.append(starts[-1] + q)
    # [batch, heads, 1, dim] of a decode step, [1, heads, tokens, dim] of a packed pass.
    return {"case": case, "query": query.unsqueeze(2) if step else query.transpose(0, 1).unsqueeze(0),
            "keys": keys, "values": values, "key_scales": key_scales, "value_scales": value_scales, "table": table,
            "contexts": torch.tensor(contexts, dtype=torch.int32, device=DEVICE),
            "starts": None if step else torch.tensor(starts, dtype=torch.int32, device=DEVICE),
            "host_contexts": tuple(contexts), "host_queries": tuple(queries)}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if kind == "append":
        return _append(state)
    return _attend(state) if kind == "attend" else _product(state)


def _held(codes, scales, dtype):
    """What a store holds, its codes times their blocks' scales, in the dtype that K and V come in."""
    blocks, heads = scales.shape
    return (codes.view(blocks, -1, heads, codes.shape[-1]) * scales[:, None, :, None]).to(dtype)


def _append(s):
    if own:
        from liteinfer_amd.rope import rope_kv_write

        q = rope_kv_write(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["slots"], s["keys"], s["values"],
                          key_scales=s["key_scales"], value_scales=s["value_scales"])
    else:
        cos, sin = s["cos"].float().unsqueeze(1), s["sin"].float().unsqueeze(1)

        def rotated(x):
            x = x.float()
            half = x.shape[-1] // 2
            return x * cos + torch.cat((-x[..., half:], x[..., :half]), dim=-1) * sin

        q = rotated(s["q"]).to(s["q"].dtype)
        slots, block = s["slots"].reshape(-1), s["case"]["block"]
        for codes, scales, rows in ((s["keys"], s["key_scales"], rotated(s["k"])),
                                    (s["values"], s["value_scales"], s["v"].float())):
            rows = rows.transpose(1, 2).reshape(slots.numel(), *codes.shape[1:])  # [tokens, heads, dim]
            at = slots // block
            # A block whose first slot is written starts anew: what it held does not count.
            anew = torch.zeros(scales.shape[0], device=DEVICE).index_add_(0, at, (slots % block == 0).float()) > 0
            old = scales.masked_fill(anew[:, None], 0.0)
            largest = torch.zeros_like(scales).index_reduce_(0, at, rows.abs().amax(dim=-1), "amax")
            new = torch.maximum(old, (largest * STEP).clamp(min=LEAST))
            # The blocks written to whose scale grows: their rows are re-expressed, then the new rows stored.
            touched = torch.zeros(scales.shape[0], dtype=torch.bool, device=DEVICE).index_fill_(0, at, True)[:, None]
            grown = (touched & (new > old))[:, None, :, None]
            held = codes.view(scales.shape[0], block, *codes.shape[1:])
            again = torch.round(held * (old * torch.reciprocal(new))[:, None, :, None])
            held.copy_(torch.where(grown, again, held))
            scales.copy_(torch.where(touched, new, scales))
            inv = torch.reciprocal(new)[at][..., None]
            codes[slots] = torch.round(rows * inv).clamp(-127, 127).to(torch.int8)
    return {"q": q, "keys": _held(s["keys"], s["key_scales"], q.dtype),
            "values": _held(s["values"], s["value_scales"], q.dtype)}


def _attend(s):
    case = s["case"]
    scaling = case["dim"] ** -0.5
    if own:
        from liteinfer_amd.attention import PagedKV, paged_attention

        kv = PagedKV(s["keys"], s["values"], s["table"], s["contexts"], query_start_loc=s["starts"],
                     max_query_len=max(s["host_queries"]), host_context_lens=s["host_contexts"],
                     host_query_lens=s["host_queries"], key_scales=s["key_scales"], value_scales=s["value_scales"])
        return paged_attention(s["query"], kv, scaling, case["groups"])
    if s["starts"] is None:
        query = s["query"].float()
        return _plain_attention(s, query, s["table"], s["contexts"], s["contexts"] - 1, scaling).to(s["query"].dtype)
    # A packed pass: the chunks, padded to the longest one, then the rows of one query each.
    chunks = case["seqs"] - case["rows"]
    query = s["query"][0].transpose(0, 1).float()  # [tokens, heads, dim]
    counts = s["starts"][1:] - s["starts"][:-1]
    out = torch.empty_like(query)
    for lo, hi in ((0, chunks), (chunks, case["seqs"])):
        if hi == lo:
            continue
        longest, widest = max(s["host_queries"][lo:hi]), max(s["host_contexts"][lo:hi])
        j = torch.arange(longest, device=DEVICE)
        there = j < counts[lo:hi, None]
        token = torch.where(there, s["starts"][lo:hi, None] + j, 0)
        first = (s["contexts"] - counts)[lo:hi]
        got = _plain_attention(s, query[token].transpose(1, 2), s["table"][lo:hi, :widest], s["contexts"][lo:hi],
                               first, scaling).transpose(1, 2)
        out[token[there]] = got[there]
    return out.to(s["query"].dtype).transpose(0, 1).unsqueeze(0)


def _plain_attention(s, query, table, contexts, first, scaling):
    """query [n, heads, queries, dim] whose first one is at position `first` [n], over the slots of `table` [n, width]."""
    case = s["case"]
    n, width = table.shape

    def rows(codes, scales):  # [n, kv heads, width, dim]
        return (codes[table] * scales[table // case["block"]][..., None]).transpose(1, 2)

    grouped = query.reshape(n, case["kv_heads"], -1, case["dim"])  # groups x queries
    scores = torch.matmul(grouped, rows(s["keys"], s["key_scales"]).transpose(2, 3)) * scaling
    scores = scores.view(n, case["kv_heads"], case["groups"], -1, width)
    key = torch.arange(width, device=DEVICE)
    position = first[:, None] + torch.arange(query.shape[2], device=DEVICE)
    seen = (key <= position[..., None]) & (key < contexts[:, None, None])
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    weights = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    total = weights.sum(dim=-1, keepdim=True)
    out = torch.matmul(weights.view(n, case["kv_heads"], -1, width), rows(s["values"], s["value_scales"]))
    return out.view(n, case["kv_heads"], case["groups"], -1, case["dim"]).div(total).reshape(query.shape)


def _product(s):
    if own:
        from liteinfer_amd.engine.ops import linear_int8

        return linear_int8(s["x"], s["codes"], s["scale"])
    x = s["x"].float()
    row_scale = (x.abs().amax(dim=1, keepdim=True) * STEP).clamp(min=LEAST)
    rows = torch.round(x * torch.reciprocal(row_scale)).clamp(-127, 127)
    return (torch.matmul(rows, s["codes"].float().t()) * row_scale * s["scale"]).to(s["x"].dtype)


# ---------------------------------------------------------------------------
# What a pass has to move and compute
# ---------------------------------------------------------------------------


def work(case):
    if case["kind"] == "product":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": 2 * m * k + k * n + 4 * n + 2 * m * n, "flops": 2 * m * k * n}
    lens = _lengths(case)
    kv_heads, dim = case["kv_heads"], case["dim"]
    heads = kv_heads * case["groups"]
    if case["kind"] == "append":
        tokens = sum(c for _, c in lens)
        blocks = sum((s + c - 1) // case["block"] - s // case["block"] + 1 for s, c in lens)
        slots = blocks * case["block"]
        # In: q, k, v, the tables, the slots, the blocks' codes and scales; out: q, and what the blocks hold.
        return {"bytes": tokens * (2 * heads * dim + 2 * kv_heads * dim + 2 * dim) * 2 + 8 * tokens
                + 2 * (blocks * kv_heads * 8 + slots * kv_heads * dim * (1 + 2)),
                "flops": 4 * tokens * (heads + 2 * kv_heads) * dim}
    queries, keys = sum(q for q, _ in lens), sum(q + p for q, p in lens)
    pairs = sum(q * p + q * (q + 1) // 2 for q, p in lens)
    return {"bytes": 2 * 2 * queries * heads * dim + 2 * keys * kv_heads * dim + 8 * keys
            + 2 * 4 * kv_heads * sum(-(-(q + p) // case["block"]) for q, p in lens),
            "flops": 4 * pairs * heads * dim}


# ---------------------------------------------------------------------------
# In 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "product": _exact_product}[case["kind"]](case, s)


def _exact_append(case, s):
    block, half = case["block"], case["dim"] // 2
    cos, sin = s["cos"].double()[:, None], s["sin"].double()[:, None]

    def turn(x):
        x = x.double()
        lo, hi = x[..., :half], x[..., half:]
        return torch.cat((lo * cos[..., :half] - hi * sin[..., :half], hi * cos[..., half:] + lo * sin[..., half:]), -1)

    found = {"q": turn(s["q"])}
    slots = s["slots"][0]
    for name, rows in (("keys", turn(s["k"])), ("values", s["v"].double())):
        codes, scales = s[name].double().unflatten(0, (-1, block)), s[name[:-1] + "_scales"].double()
        rows = rows.permute(0, 2, 1, 3).flatten(0, 1)
        # Every row of every block beside the new rows that fall into it.
        new = torch.zeros_like(codes).flatten(0, 1)
        new[slots] = rows
        written = torch.zeros(new.shape[0], dtype=torch.bool, device=DEVICE)
        written[slots] = True
        new, written = new.view_as(codes), written.view(-1, block)
        touched = written.any(dim=1)[:, None]
        kept = torch.where(written[:, :1], 0.0, scales)
        largest = new.abs().amax(dim=(1, 3)) / 127
        grown = torch.where(touched, torch.maximum(kept, largest.clamp(min=LEAST)), scales)
        moved = touched & (grown > kept)
        before = torch.where(moved[:, None, :, None], torch.round(codes * (kept / grown)[:, None, :, None]), codes)
        # grown is zero only for blocks that nothing was written to.
        at = torch.where(grown > 0, grown, 1.0)[:, None, :, None]
        after = torch.where(written[:, :, None, None], torch.round(new / at).clamp(-127, 127), before)
        found[name] = after * grown[:, None, :, None]
    return found


def _exact_attend(case, s):
    query = s["query"][:, :, 0] if s["starts"] is None else s["query"][0].transpose(0, 1)  # [tokens, heads, dim]
    out = torch.empty(query.shape, dtype=torch.float64, device=DEVICE)
    at = 0
    for i, (nq, ctx) in enumerate(zip(s["host_queries"], s["host_contexts"])):
        slots = s["table"][i, :ctx]
        key = s["keys"][slots].double() * s["key_scales"][slots // case["block"]].double()[..., None]
        value = s["values"][slots].double() * s["value_scales"][slots // case["block"]].double()[..., None]
        hidden = torch.arange(ctx, device=DEVICE) > torch.arange(ctx - nq, ctx, device=DEVICE)[:, None]
        for h in range(case["kv_heads"]):
            q = query[at:at + nq, h * case["groups"]:(h + 1) * case["groups"]].double().transpose(0, 1)
            score = (q.reshape(-1, case["dim"]) @ key[:, h].t()).view(case["groups"], nq, ctx) / math.sqrt(case["dim"])
            share = torch.softmax(score.masked_fill(hidden, float("-inf")), dim=-1)
            got = (share.view(-1, ctx) @ value[:, h]).view(case["groups"], nq, case["dim"])
            out[at:at + nq, h * case["groups"]:(h + 1) * case["groups"]] = got.transpose(0, 1)
        at += nq
    return out.unsqueeze(2) if s["starts"] is None else out.transpose(0, 1).unsqueeze(0)


def _exact_product(case, s):
    x = s["x"].double()
    scale = x.abs().max(dim=1).values / 127
    scale = scale.clamp(min=LEAST)
    codes = (x / scale[:, None]).round().clamp(-127, 127)
    return (codes @ s["codes"].double().t()) * scale[:, None] * s["scale"].double()
