"""The operators of a bounded cache, as cases to be timed and compared.

A request that generates for a long time keeps its cost per token bounded in one
of two ways.  It attends its newest tokens and a few first ones only (``window``),
or it attends all that its cache holds, adds up the attention that each cached
token receives (``scored``), and now and then gives up the tokens that received
least (``evict``).  K/V, queries, scores and block tables are drawn from the seed;
blocks are handed out in random order, as a cache that has been serving for a
while holds them.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_INDEX = {"int32": torch.int32, "int64": torch.int64}
_MAX_KV_BYTES = 700 << 20  # of a drawn case: under the largest listed one's


# ------------------------------------------------------------------ cases --
def _case(kind, name=None, **over):
    case = {"kind": kind, "batch": 8, "ctx": 2048, "lengths": "full", "q_heads": 16, "kv_heads": 2, "head_dim": 128,
            "block": 32, "dtype": "bf16", "index": "int32"}
    case.update(over)
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # The first answer tokens of one short chat: everything is visible, and the call is all latency.
        _case("window", "window-first-tokens", batch=1, ctx=100, window=128, sinks=4, block=16),
        # Eight chats in a model with a window of 1024.
        _case("window", "window-chat", window=1024, sinks=4),
        # A long-document server: the blocks that left the window have gone back to the pool.  The largest window.
        _case("window", "window-documents", batch=64, ctx=32768, lengths="half", q_heads=32, kv_heads=8, window=4096,
              sinks=64),
        # Small heads, seven query heads for each KV head, an odd window that ends inside blocks, rows of very
        # different lengths, 64-bit indices.
        _case("window", "window-head64", batch=48, ctx=8192, lengths="log", q_heads=14, head_dim=64, dtype="fp16",
              block=8, window=1000, sinks=5, index="int64"),
        # One short chat that will be pruned later.
        _case("scored", "scored-first-tokens", batch=1, ctx=300, block=16),
        # Eight chats at their budget.
        _case("scored", "scored-chat"),
        # A serving batch somewhere between an eviction and the next: the largest.
        _case("scored", "scored-serving", batch=32, ctx=8192, lengths="half", q_heads=32, kv_heads=8),
        # Rows of very different lengths, small heads.
        _case("scored", "scored-mixed", batch=16, ctx=32768, lengths="log", q_heads=14, head_dim=64, dtype="fp16",
              block=16, index="int64"),
        # One chat that passed its budget by a quarter.
        _case("evict", "evict-one-chat", batch=1, ctx=640, keep=512, sinks=4, recent=64, block=16),
        # Eight chats cut to half.
        _case("evict", "evict-chat", keep=1024, sinks=4, recent=256),
        # A serving batch under memory pressure; some rows are within their budget already.
        _case("evict", "evict-serving", batch=32, ctx=4096, lengths="half", q_heads=32, kv_heads=8, keep=2500, sinks=16,
              recent=512),
        # Two long documents cut to a quarter after they have been read, small heads.
        _case("evict", "evict-documents", batch=2, ctx=32768, q_heads=32, kv_heads=8, head_dim=64, dtype="fp16",
              keep=8192, sinks=4, recent=1024, index="int64"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("window", "scored", "evict"))
    head_dim = rng.choice((128, 128, 128, 64))
    if head_dim == 64:
        q_heads, kv_heads = rng.choice(((14, 2), (16, 2), (32, 8), (71, 1)))
    else:
        q_heads, kv_heads = rng.choice(((16, 2), (16, 2), (32, 8), (32, 8), (16, 1), (16, 16), (12, 4)))
    token = kv_heads * head_dim * 4  # bytes of one token's K and V
    batch = _log_int(rng, 1, 128)
    over = {"batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "block": rng.choice((8, 16, 32, 32)), "dtype": rng.choice(("bf16", "bf16", "fp16")),
            "index": rng.choice(("int32", "int64")), "lengths": rng.choice(("full", "half", "half", "log"))}
    if kind == "window":
        sinks = rng.choice((0, 1, 4, 4, 37))
        window = _log_int(rng, 16, max(17, min(8192, _MAX_KV_BYTES // (batch * token) - sinks)))
        return _case(kind, ctx=_log_int(rng, 64, 65536), window=window, sinks=sinks, **over)
    # query heads of large groups cost more than their K/V
    most = min(32768, _MAX_KV_BYTES // (batch * token * (2 if q_heads > 16 * kv_heads else 1)))
    if kind == "scored":
        return _case(kind, ctx=_log_int(rng, 32, max(33, most)), **over)
    ctx = _log_int(rng, 128, max(129, most // 2))
    keep = max(16, int(ctx * rng.uniform(0.1, 1.0)))
    return _case(kind, ctx=ctx, keep=keep, sinks=rng.choice((0, 4, 13)), recent=rng.randrange(0, keep - 13), **over)


# ----------------------------------------------------------------- inputs --
def _lengths(case, seed):
    """Tokens of each row.  Half: between half of ctx and ctx; log: spread evenly over the logarithm from
    ctx / 256 to ctx.  The lengths' sum is close to the same for every seed."""
    n, ctx = case["batch"], case["ctx"]
    if case["lengths"] == "full":
        return [ctx] * n
    rng = random.Random(seed)
    at = [(i + rng.random()) / n for i in range(n)]  # one from each n-th of the range
    rng.shuffle(at)
    low = max(1, ctx // 2 if case["lengths"] == "half" else ctx // 256)
    if case["lengths"] == "half":
        return [min(ctx, int(low + u * (ctx + 1 - low))) for u in at]
    return [max(1, min(ctx, int(round(low * (ctx / low) ** u)))) for u in at]


def _tables(case, lens, gen):
    """(block table, wide enough for ctx tokens, number of blocks): -1 past each row's blocks, and for a
    window also where no visible token lies, as those blocks belong to others by now."""
    block = case["block"]
    need = [-(-n // block) for n in lens]
    held = [torch.ones(n, dtype=torch.bool) for n in need]
    if case["kind"] == "window":
        for n, row in zip(lens, held):
            row[-(-case["sinks"] // block) : max(0, n - case["window"]) // block] = False
    total = sum(int(row.sum()) for row in held)
    if case["kind"] == "evict":  # a pool that holds every row at its longest
        total = len(lens) * -(-case["ctx"] // block)
    order = torch.randperm(total, device="cuda", generator=gen).cpu()
    table = torch.full((len(lens), -(-case["ctx"] // block)), -1, dtype=torch.int64)
    at = 0
    for b, row in enumerate(held):
        count = int(row.sum())
        table[b, : row.numel()][row] = order[at : at + count]
        at += count
    return table, total


def _normal(shape, dtype, gen, std=1.0):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    kind, dtype, hkv, d = case["kind"], _DTYPES[case["dtype"]], case["kv_heads"], case["head_dim"]
    lens = _lengths(case, seed)
    table, blocks = _tables(case, lens, gen)
    index = _INDEX[case["index"]]
    state = {"case": case, "tables": table.to("cuda", index), "lens": torch.tensor(lens, device="cuda", dtype=index),
             "k": _normal((blocks, hkv, case["block"], d), dtype, gen),
             "v": _normal((blocks, hkv, case["block"], d), dtype, gen)}
    rows, tokens = len(lens), table.shape[1] * case["block"]
    if kind != "evict":
        # queries of twice unit size: scores spread as a trained head's do, a few tokens weighing most
        state["q"] = _normal((rows, case["q_heads"], d), dtype, gen, 2.0)
        state["out"] = torch.empty_like(state["q"])
    if kind != "window":
        # weight gathered so far: a heavy tail, and tokens that no query has looked at
        scores = torch.exp(_normal((rows, hkv, tokens), torch.float32, gen, 1.5))
        scores *= torch.rand((rows, hkv, tokens), device="cuda", generator=gen) < 0.9
        past = torch.arange(tokens, device="cuda") >= state["lens"][:, None]
        state["scores"] = scores.masked_fill_(past[:, None], 0.0)
    if kind == "evict":
        # the table of the next stretch: a server keeps two and takes them in turn
        state["next_scores"] = torch.zeros_like(scores)
        state["kept"] = torch.empty((rows, hkv, case["keep"]), device="cuda", dtype=torch.int32)
        state["next_lens"] = torch.empty_like(state["lens"])
    return state


# -------------------------------------------------------------------- run --
def run(state):
    case = state["case"]
    return _run_own(state) if own else {"window": _window, "scored": _scored, "evict": _evict}[case["kind"]](state)


def _run_own(state):
    import flashdec_amd as fd

    case = state["case"]
    k, v, tables, lens = state["k"], state["v"], state["tables"], state["lens"]
    if case["kind"] == "window":
        return fd.paged_decode_attention_window_into(state["q"], k, v, tables, lens, state["out"], case["window"],
                                                     sink_tokens=case["sinks"])
    if case["kind"] == "scored":
        out = fd.paged_decode_attention_scored_into(state["q"], k, v, tables, lens, state["out"], state["scores"])
        return {"out": out, "scores": state["scores"]}
    fd.paged_kv_evict_into(k, v, tables, lens, state["scores"], case["keep"], state["kept"], state["next_lens"],
                           sink_tokens=case["sinks"], recent_tokens=case["recent"], new_scores=state["next_scores"])
    return {"kept": state["kept"], "lens": state["next_lens"], "scores": state["next_scores"], "k": k, "v": v}


def _gather(cache, tables, tokens):
    """float32 rows [B, Hkv, n, D] of the tokens [B, n] (those without a block read block 0)."""
    block = cache.shape[2]
    ids = tables.long().gather(1, tokens // block).clamp_min(0)
    return cache[ids, :, tokens % block].float().permute(0, 2, 1, 3).contiguous()


def _attend(q, keys, values, visible):
    """Attention of q [B, Hq, D] on rows [B, Hkv, n, D] where visible [B, n], in 32 bits: (out, weights
    [B, Hkv, n, G])."""
    rows, hkv, _, d = keys.shape
    heads = q.float().view(rows, hkv, -1, d).transpose(2, 3).contiguous()
    s = (keys @ heads) / math.sqrt(d)  # [B, Hkv, n, G]
    s = s.masked_fill(~visible[:, None, :, None], -math.inf)
    p = torch.exp(s - s.amax(dim=2, keepdim=True))
    p = p / p.sum(dim=2, keepdim=True)
    out = p.transpose(2, 3).contiguous() @ values
    return out.reshape(q.shape).to(q.dtype), p


def _window(state):
    case, lens = state["case"], state["lens"].long()
    sinks, window = case["sinks"], case["window"]
    # the sinks, then the window's tokens, each token once
    at = torch.arange(sinks + window, device=lens.device)
    start = (lens - window).clamp_min(sinks)[:, None]
    tokens = torch.where(at < sinks, at, start + at - sinks)
    visible = tokens < lens[:, None]
    tokens = torch.minimum(tokens, lens[:, None] - 1)
    keys, values = (_gather(state[c], state["tables"], tokens) for c in ("k", "v"))
    return _attend(state["q"], keys, values, visible)[0]


def _scored(state):
    lens = state["lens"].long()
    at = torch.arange(state["scores"].shape[2], device=lens.device)
    visible = at < lens[:, None]
    tokens = torch.minimum(at, lens[:, None] - 1)
    keys, values = (_gather(state[c], state["tables"], tokens) for c in ("k", "v"))
    out, weights = _attend(state["q"], keys, values, visible)
    state["scores"] += weights.sum(dim=3)
    return {"out": out, "scores": state["scores"]}


def _evict(state):
    case, lens, scores = state["case"], state["lens"].long(), state["scores"]
    keep, block = case["keep"], case["block"]
    at = torch.arange(scores.shape[2], device=lens.device)
    live = (at < lens[:, None])[:, None]
    always = (live & ((at < case["sinks"]) | (at >= lens[:, None] - case["recent"])[:, None]))
    rank = torch.where(always, math.inf, scores).masked_fill(~live, -math.inf)
    best = torch.sort(rank, dim=2, descending=True, stable=True).indices[:, :, :keep]
    if best.shape[2] < keep:  # the tables hold fewer tokens than may be kept
        best = torch.nn.functional.pad(best, (0, keep - best.shape[2]), value=scores.shape[2])
    best = torch.where(best < lens[:, None, None], best, torch.iinfo(torch.int32).max)
    kept = best.sort(dim=2).values
    n = lens.clamp_max(keep)
    # entries behind a row's last one repeat it: the same values to the same place
    to = torch.minimum(torch.arange(keep, device=lens.device), n[:, None] - 1)
    source = kept.gather(2, to[:, None].expand_as(kept))
    head = torch.arange(scores.shape[1], device=lens.device)[None, :, None]
    row = torch.arange(scores.shape[0], device=lens.device)[:, None, None]
    tables = state["tables"].long()
    to = to[:, None].expand_as(kept)
    for cache in (state["k"], state["v"]):
        moved = cache[tables[row, source // block], head, source % block]
        cache[tables[row, to // block], head, to % block] = moved
    moved = scores[row, head, source]
    state["next_scores"].masked_fill_(live, 0.0)
    state["next_scores"][row, head, to] = moved
    state["kept"].copy_(torch.where(kept < lens[:, None, None], kept, -1))
    state["next_lens"].copy_(n)
    return {"kept": state["kept"], "lens": state["next_lens"], "scores": state["next_scores"], "k": state["k"],
            "v": state["v"]}


# ------------------------------------------------------------------- work --
def work(case):
    hq, hkv, d, rows = case["q_heads"], case["kv_heads"], case["head_dim"], case["batch"]
    lens = _lengths(case, 0)
    tokens = sum(lens)
    if case["kind"] == "evict":
        # scores read and written, the list, and K/V read and written of the kept tokens behind the first that
        # goes (of rows over their budget)
        kept = sum(min(n, case["keep"]) for n in lens)
        moved = sum(max(0, case["keep"] - case["sinks"]) for n in lens if n > case["keep"])
        return {"bytes": hkv * (8 * tokens + 4 * kept + 8 * moved * d), "flops": hkv * tokens}
    if case["kind"] == "window":
        tokens = sum(min(n, case["sinks"] + case["window"]) for n in lens)
    table = 8 * tokens * hkv if case["kind"] == "scored" else 0
    return {"bytes": tokens * hkv * d * 4 + rows * hq * d * 4 + table, "flops": tokens * hq * d * 4}


# ------------------------------------------------------------------ exact --
def exact(case, seed):
    """Row by row from the definitions, in 64 bits."""
    state = prepare(case, seed)
    tables, lens = state["tables"].long().cpu(), state["lens"].tolist()
    if case["kind"] == "evict":
        return _exact_evict(case, state, tables, lens)
    hkv, block = case["kv_heads"], case["block"]
    group = case["q_heads"] // hkv
    scale = 1.0 / math.sqrt(case["head_dim"])
    outs = []
    for b, n in enumerate(lens):
        seen = torch.arange(n)
        if case["kind"] == "window":
            seen = seen[(seen < case["sinks"]) | (seen >= n - case["window"])]
        ids, off = tables[b, seen // block].cuda(), (seen % block).cuda()
        for h in range(hkv):
            keys, values = (state[c][ids, h, off].double() for c in ("k", "v"))
            query = state["q"][b, h * group : (h + 1) * group].double()
            p = torch.softmax(torch.mm(query, keys.t().contiguous()) * scale, dim=1)
            outs.append(torch.mm(p, values))
            if case["kind"] == "scored":
                total = state["scores"][b, h, :n].double() + p.sum(dim=0)
                state.setdefault("exact", []).append(torch.nn.functional.pad(total, (0, state["scores"].shape[2] - n)))
    out = torch.cat(outs).view(state["q"].shape)
    if case["kind"] == "window":
        return out
    return {"out": out, "scores": torch.stack(state["exact"]).view(state["scores"].shape)}


def _exact_evict(case, state, tables, lens):
    block, keep, hkv = case["block"], case["keep"], case["kv_heads"]
    scores = state["scores"].cpu().double()
    new_scores = torch.zeros_like(scores)
    kept = torch.full((len(lens), hkv, keep), -1, dtype=torch.int32)
    caches = [state["k"].clone(), state["v"].clone()]
    for b, n in enumerate(lens):
        for h in range(hkv):
            stay = list(range(n))
            if n > keep:
                inner = list(range(case["sinks"], n - case["recent"]))
                value = scores[b, h].tolist()
                inner.sort(key=lambda t: (-value[t], t))
                stay = sorted([*range(case["sinks"]), *inner[: keep - case["sinks"] - case["recent"]],
                               *range(n - case["recent"], n)])
            at = torch.tensor(stay, dtype=torch.int64)
            kept[b, h, : len(stay)] = at.int()
            new_scores[b, h, : len(stay)] = scores[b, h, at]
            to = torch.arange(len(stay))
            source, off = tables[b, at // block].cuda(), (at % block).cuda()
            place, there = tables[b, to // block].cuda(), (to % block).cuda()
            for new, name in zip(caches, ("k", "v")):
                new[place, h, there] = state[name][source, h, off]
    device = state["k"].device
    return {"kept": kept.to(device), "lens": torch.tensor([min(n, keep) for n in lens], device=device),
            "scores": new_scores.to(device), "k": caches[0], "v": caches[1]}
