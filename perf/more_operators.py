"""The operators of long contexts, as cases to be timed and compared.

A long context costs decode its bytes.  It costs fewer where the cache holds keys
and values in 4 bits (``append``: new tokens are rotated, quantised and stored;
``fp4``: decode over such a cache), or where each KV head attends the blocks that
matter to its queries only (``bounds``: the smallest and largest key of every
complete block; ``sparse``: blocks chosen by them, and attention on the chosen
ones).  Inputs are drawn from the seed; blocks are handed out in random order, as a
cache that has been serving for a while holds them.

The 4-bit format: 32 neighbouring dims of a token's head share a power of two, held
as its exponent plus 127 in one byte, and each is the nearest of 0, 1/2, 1, 3/2, 2,
3, 4, 6 and their negatives times it.  A block of one KV head holds its tokens'
codes, two a byte, and behind them their scale bytes: of keys token by token, of
values four tokens at a time, for each the codes of a sixteenth of the dims, and
the scale bytes of the same 32 dims.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_INDEX = {"int32": torch.int32, "int64": torch.int64}
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_MAX_FP4_BYTES = 500 << 20  # K and V of a drawn fp4 case: under the largest listed one's, as the others
_MAX_KEY_BYTES = 250 << 20
_MAX_SPARSE_BYTES = 300 << 20
_MAX_APPEND_TOKENS = 8000


# ------------------------------------------------------------------ cases --
def _case(kind, name=None, **over):
    case = {"kind": kind, "batch": 8, "ctx": 2048, "lengths": "full", "q_heads": 16, "kv_heads": 2, "head_dim": 128,
            "block": 32, "dtype": "bf16", "index": "int32"}
    case.update(over)
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # The next token of one chat.
        _case("append", "append-one-token", batch=1, ctx=100, new=1, rotary=128, block=16),
        # Pieces of seven prompts of a model with small heads of which half is rotated, 64-bit indices.
        _case("append", "append-pieces", batch=7, ctx=900, new=111, lengths="half", q_heads=14, head_dim=64, rotary=32,
              dtype="fp16", block=8, index="int64"),
        # Long prompts on their way into the cache: the most tokens.
        _case("append", "append-prompts", batch=4, ctx=8192, new=2048, lengths="half", q_heads=32, kv_heads=8,
              rotary=128),
        # The first answer tokens of one short chat: the call is all latency.
        _case("fp4", "fp4-first-tokens", batch=1, ctx=100, block=16),
        # Eight chats.
        _case("fp4", "fp4-chat"),
        # Rows of very different lengths, small heads, seven query heads for each KV head.
        _case("fp4", "fp4-mixed", batch=16, ctx=32768, lengths="log", q_heads=14, head_dim=64, dtype="fp16", block=16,
              index="int64"),
        # A full serving batch: the most bytes.
        _case("fp4", "fp4-serving", batch=64, ctx=8192, q_heads=32, kv_heads=8),
        # A serving batch after eight steps: the blocks that they completed, in about every fourth row.
        _case("bounds", "bounds-steps", batch=64, ctx=8192, lengths="half", new=8, q_heads=32, kv_heads=8),
        # Four long documents after they have been read.
        _case("bounds", "bounds-documents", batch=4, ctx=32768, lengths="half", new=32768, q_heads=32, kv_heads=8),
        # One chat with a few pages of context.
        _case("sparse", "sparse-chat", batch=1, ctx=8192, select=32, sinks=1, recent=2),
        # Rows of very different lengths, the shortest with fewer blocks than are chosen, small heads.
        _case("sparse", "sparse-mixed", batch=8, ctx=65536, lengths="log", select=100, sinks=1, recent=3, q_heads=14,
              head_dim=64, dtype="fp16", block=16, index="int64"),
        # A long-document server: an eighth to a quarter of each row is attended.
        _case("sparse", "sparse-documents", batch=16, ctx=32768, lengths="half", select=128, sinks=1, recent=4,
              q_heads=32, kv_heads=8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo + 1, hi))))))


def draw(rng):
    kind = rng.choice(("append", "fp4", "bounds", "sparse"))
    head_dim = rng.choice((128, 128, 128, 64))
    if head_dim == 64:
        q_heads, kv_heads = rng.choice(((14, 2), (16, 2), (32, 8), (71, 1)))
    else:
        q_heads, kv_heads = rng.choice(((16, 2), (16, 2), (32, 8), (32, 8), (16, 1), (16, 16), (12, 4)))
    batch = _log_int(rng, 1, 128)
    over = {"batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "block": rng.choice((8, 16, 32, 32)), "dtype": rng.choice(("bf16", "bf16", "fp16")),
            "index": rng.choice(("int32", "int64")), "lengths": rng.choice(("full", "half", "half", "log"))}
    elements = batch * kv_heads * head_dim  # of one token in every row
    if kind == "append":
        most = max(1, _MAX_APPEND_TOKENS * 32 // (batch * max(q_heads, 32)))
        new = rng.choice((1, _log_int(rng, 1, most)))
        rotary = rng.choice((head_dim, head_dim, head_dim // 2))
        return _case(kind, new=new, ctx=new + _log_int(rng, 1, 8192), rotary=rotary, **over)
    if kind == "fp4":
        # query heads of large groups cost more than their K/V
        most = _MAX_FP4_BYTES * 16 // (elements * 17 * (2 if q_heads > 16 * kv_heads else 1))
        return _case(kind, ctx=_log_int(rng, 1, min(65536, most)), **over)
    if kind == "bounds":
        ctx = _log_int(rng, 16, min(65536, _MAX_KEY_BYTES // (elements * 2)))
        return _case(kind, ctx=ctx, new=rng.choice((1, 1, _log_int(rng, 1, ctx), ctx)), **over)
    ctx = _log_int(rng, 64, min(131072, _MAX_SPARSE_BYTES // (elements * 2)))
    sinks, recent = rng.choice((0, 1, 1, 3)), rng.choice((1, 2, 5))
    most = min(ctx, _MAX_SPARSE_BYTES // (elements * 4)) // over["block"]
    return _case(kind, ctx=ctx, select=sinks + recent + _log_int(rng, 1, max(2, most // 2)), sinks=sinks, recent=recent,
                 **over)


# ----------------------------------------------------------------- inputs --
def _lengths(case, seed):
    """Tokens of each row.  Half: between half of ctx and ctx; log: spread evenly over the logarithm from
    ctx / 256 to ctx.  The lengths' sum is close to the same for every seed."""
    n, ctx = case["batch"], case["ctx"]
    low = max(1, ctx // 2 if case["lengths"] == "half" else ctx // 256)
    if case["kind"] == "append":
        low = max(low, case["new"])
    if case["lengths"] == "full":
        return [ctx] * n
    rng = random.Random(seed)
    at = [(i + rng.random()) / n for i in range(n)]  # one from each n-th of the range
    rng.shuffle(at)
    if case["lengths"] == "half":
        return [min(ctx, int(low + u * (ctx + 1 - low))) for u in at]
    return [max(low, min(ctx, int(round(low * (ctx / low) ** u)))) for u in at]


def _tables(case, lens, gen):
    """(block table, wide enough for ctx tokens, -1 past each row's blocks; number of blocks)."""
    need = [-(-n // case["block"]) for n in lens]
    table = torch.full((len(lens), -(-case["ctx"] // case["block"])), -1, dtype=torch.int64)
    total = sum(need)
    if case["kind"] == "bounds":  # a pool that holds every row at its longest
        total = table.numel()
    order = torch.randperm(total, device="cuda", generator=gen).cpu()
    for b, row in enumerate(order[: sum(need)].split(need)):
        table[b, : row.numel()] = row
    return table, total


def _normal(shape, dtype, gen, std=1.0):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=gen)


def _pool(blocks, case, gen, values):
    """A 4-bit pool [blocks, kv_heads, bytes of a block] of normal keys or values, quantised some blocks at a time."""
    heads, block, d = case["kv_heads"], case["block"], case["head_dim"]
    pool = torch.empty((blocks, heads, block * d * 17 // 32), device="cuda", dtype=torch.uint8)
    step = max(1, (32 << 20) // (heads * block * d))
    for at in range(0, blocks, step):
        part = pool[at : at + step]
        x = _normal((part.shape[0], heads, block, d), torch.float32, gen)
        for plane, held in zip(_planes(part, case, values), _quantise(x)):
            plane.copy_(held.view(plane.shape))
    return pool


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    kind, dtype, hkv, d = case["kind"], _DTYPES[case["dtype"]], case["kv_heads"], case["head_dim"]
    lens = _lengths(case, seed)
    table, blocks = _tables(case, lens, gen)
    index = _INDEX[case["index"]]
    rows, block = len(lens), case["block"]
    state = {"case": case, "tables": table.to("cuda", index), "lens": torch.tensor(lens, device="cuda", dtype=index)}
    if kind == "append":
        # each row's last `new` tokens; a cos/sin table of the positions, as a model keeps one
        new, half = case["new"], case["rotary"] // 2
        at = torch.stack([torch.arange(n - new, n) for n in lens])
        state["positions"] = at.flatten().to("cuda", index)
        state["block_ids"] = table.gather(1, at // block).flatten().to("cuda", index)
        state["block_offsets"] = (at % block).flatten().to("cuda", index)
        angles = torch.arange(case["ctx"]).double()[:, None] * 10000.0 ** (-torch.arange(half).double() / half)
        state["cos_sin"] = torch.stack((angles.cos(), angles.sin())).to("cuda", torch.float32).contiguous()
        for name, heads in (("q", case["q_heads"]), ("k", hkv), ("v", hkv)):
            state[name] = _normal((rows * new, heads, d), dtype, gen)
        shape = (blocks, hkv, block * d * 17 // 32)
        state["k_cache"], state["v_cache"] = (torch.zeros(shape, device="cuda", dtype=torch.uint8) for _ in range(2))
        state["q_out"] = torch.empty_like(state["q"])
        state["k_out"], state["v_out"] = torch.empty_like(state["k"]), torch.empty_like(state["v"])
        return state
    if kind == "fp4":
        state["k_cache"], state["v_cache"] = _pool(blocks, case, gen, False), _pool(blocks, case, gen, True)
    else:
        state["k_cache"] = _normal((blocks, hkv, block, d), dtype, gen)
        # bounds of every block but those that `new` tokens may have completed, which a server finds stale
        state["bounds"] = torch.stack((state["k_cache"].amin(dim=2), state["k_cache"].amax(dim=2)), dim=2)
    if kind == "bounds":
        b = torch.arange(table.shape[1])
        done = torch.tensor(lens)[:, None] // block
        fresh = (b < done) & (b >= (torch.tensor(lens)[:, None] - case["new"]).clamp_min(0) // block)
        state["bounds"][table[fresh].cuda()] = 0
        return state
    # queries of twice unit size: scores spread as a trained head's do, a few tokens weighing most
    state["q"] = _normal((rows, case["q_heads"], d), dtype, gen, 2.0)
    state["out"] = torch.empty_like(state["q"])
    if kind == "sparse":
        state["v_cache"] = _normal((blocks, hkv, block, d), dtype, gen)
        state["blocks"] = torch.empty((rows, hkv, case["select"]), device="cuda", dtype=torch.int32)
        state["head_tables"] = torch.empty_like(state["blocks"])
        state["head_lens"] = torch.empty((rows, hkv), device="cuda", dtype=torch.int32)
    return state


# -------------------------------------------------------------------- run --
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state)
    return {"append": _append, "fp4": _fp4, "bounds": _bounds, "sparse": _sparse}[kind](state)


def _run_own(state):
    import flashdec_amd as fd

    case, tables, lens, k, v = (state.get(x) for x in ("case", "tables", "lens", "k_cache", "v_cache"))
    if case["kind"] == "append":
        ids, offsets = state["block_ids"], state["block_offsets"]
        fd.fused_rope_kv_append_fp4(state["q"], state["k"], state["v"], k, v, ids, offsets, state["positions"],
                                    rotary_dim=case["rotary"], cos_sin_table=state["cos_sin"], q_out=state["q_out"],
                                    check_indices=False)
        fd.paged_kv_read_fp4_into(k, v, ids, offsets, state["k_out"], state["v_out"])
        return {"q": state["q_out"], "k": state["k_out"], "v": state["v_out"]}
    if case["kind"] == "fp4":
        return fd.paged_decode_attention_fp4_into(state["q"], k, v, tables, lens, state["out"])
    if case["kind"] == "bounds":
        return fd.paged_key_bounds(k, tables, lens, state["bounds"], new_tokens=case["new"])
    chosen = fd.paged_block_select_into(state["q"], k, state["bounds"], tables, lens, state["blocks"],
                                        state["head_tables"], state["head_lens"], sink_blocks=case["sinks"],
                                        recent_blocks=case["recent"])
    out = fd.paged_decode_attention_blocks_into(state["q"], k, v, chosen, state["out"])
    return {"out": out, "blocks": chosen.blocks}


def _quantise(x):
    """(codes, scale bytes) of float32 [..., D], 32 dims a scale: the least power of two that leaves the group's
    largest at 7 or below, so that none is further from its level than half of the widest step."""
    groups = x.unflatten(-1, (-1, 32))
    bits = groups.abs().amax(dim=-1).view(torch.int32)
    byte = (((bits + 0x1FFFFF) >> 23) - 2).clamp(2, 252)
    y = groups / (byte << 23).view(torch.float32)[..., None]
    a, code = y.abs(), torch.zeros_like(y, dtype=torch.uint8)
    code += (a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte()  # ties to the even code
    code += (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5.0).byte()
    code += torch.signbit(y).byte() * 8
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.byte()


def _values(codes, scales):
    """float32 [..., D] of codes [..., D / 2] and scale bytes [..., D / 32]."""
    levels = torch.tensor(_LEVELS + tuple(-x for x in _LEVELS), device=codes.device)
    x = torch.stack((levels[(codes & 15).int()], levels[(codes >> 4).int()]), dim=-1).flatten(-2)
    return (x.unflatten(-1, (-1, 32)) * (scales.int() << 23).view(torch.float32)[..., None]).flatten(-2)


def _planes(pool, case, values):
    """Views of a 4-bit pool: codes [blocks, heads, block / 4, 4, 16, D / 32] and scale bytes
    [blocks, heads, block / 4, 4, D / 32]."""
    block, d = case["block"], case["head_dim"]
    codes, scales = pool[..., : block * d // 2], pool[..., block * d // 2 :]
    if values:
        return (codes.unflatten(-1, (block // 4, 16, 4, d // 32)).transpose(-3, -2),
                scales.unflatten(-1, (block // 4, d // 32, 4)).transpose(-2, -1))
    return codes.unflatten(-1, (block // 4, 4, 16, d // 32)), scales.unflatten(-1, (block // 4, 4, d // 32))


def _rotate(x, cos, sin, rotary):
    half = rotary // 2
    x1, x2, rest = x[..., :half], x[..., half:rotary], x[..., rotary:]
    return torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin, rest), dim=-1)


def _append(state):
    case, at = state["case"], state["positions"].long()
    cos, sin = (plane[at][:, None] for plane in state["cos_sin"])
    state["q_out"].copy_(_rotate(state["q"].float(), cos, sin, case["rotary"]))
    keys = _rotate(state["k"].float(), cos, sin, case["rotary"])
    ids, offsets = state["block_ids"].long(), state["block_offsets"].long()
    where = ids, slice(None), offsets // 4, offsets % 4
    for x, pool, out, values in ((keys, "k_cache", "k_out", False), (state["v"].float(), "v_cache", "v_out", True)):
        codes, scales = _planes(state[pool], case, values)
        new, scales[where] = _quantise(x)
        codes[where] = new.unflatten(-1, codes.shape[-2:])
        state[out].copy_(_values(codes[where].flatten(-2), scales[where]))
    return {"q": state["q_out"], "k": state["k_out"], "v": state["v_out"]}


def _attend(q, keys, values, visible):
    """Attention of q [B, Hq, D] on rows [B, Hkv, n, D] where visible [B, 1 or Hkv, n], in 32 bits."""
    rows, hkv, _, d = keys.shape
    heads = q.float().view(rows, hkv, -1, d).transpose(2, 3).contiguous()
    s = (keys @ heads) / math.sqrt(d)  # [B, Hkv, n, G]
    s = s.masked_fill(~visible[..., None], -math.inf)
    p = torch.exp(s - s.amax(dim=2, keepdim=True))
    p = p / p.sum(dim=2, keepdim=True)
    return (p.transpose(2, 3).contiguous() @ values).reshape(q.shape).to(q.dtype)


def _fp4(state):
    case, tables, lens = state["case"], state["tables"].long().clamp_min(0), state["lens"].long()
    rows = []
    for name, values in (("k_cache", False), ("v_cache", True)):
        codes, scales = (x[tables].transpose(1, 2).flatten(2, 4) for x in _planes(state[name], case, values))
        rows.append(_values(codes.flatten(-2), scales))  # [B, Hkv, n, D]
    at = torch.arange(rows[0].shape[2], device=lens.device)
    return _attend(state["q"], *rows, (at < lens[:, None])[:, None])


def _bounds(state):
    case, tables, lens, bounds = state["case"], state["tables"].long(), state["lens"].long()[:, None], state["bounds"]
    b = torch.arange(tables.shape[1], device=lens.device)
    first = (lens - case["new"]).clamp_min(0) // case["block"]
    ids = tables[(b < lens // case["block"]) & (b >= first)]
    keys = state["k_cache"][ids].float()
    bounds[ids] = torch.stack((keys.amin(dim=2), keys.amax(dim=2)), dim=2).to(bounds.dtype)
    return bounds


def _sparse(state):
    case, lens, tables = state["case"], state["lens"].long(), state["tables"].long()
    block, select = case["block"], case["select"]
    rows, hkv, d = len(lens), case["kv_heads"], case["head_dim"]
    q = state["q"].double().view(rows, 1, hkv, -1, d)
    up, down = q.clamp_min(0).sum(dim=3), q.clamp_max(0).sum(dim=3)
    held = state["bounds"][tables.clamp_min(0)].double()  # [B, n, Hkv, 2, D]
    score = (up * held[:, :, :, 1] + down * held[:, :, :, 0]).sum(dim=-1).float().transpose(1, 2)
    b = torch.arange(tables.shape[1], device=lens.device)
    count = -(-lens // block)[:, None]
    always = ((b < case["sinks"]) | (b >= count - case["recent"]))[:, None]
    rank = torch.where(always, math.inf, score).masked_fill((b >= count)[:, None], -math.inf)
    best = torch.sort(rank, dim=2, descending=True, stable=True).indices[:, :, :select]
    if best.shape[2] < select:  # the tables hold fewer blocks than may be chosen
        best = torch.nn.functional.pad(best, (0, select - best.shape[2]), value=tables.shape[1])
    best = torch.where(best < count[:, :, None], best, torch.iinfo(torch.int32).max).sort(dim=2).values
    there = best < count[:, :, None]
    state["blocks"].copy_(torch.where(there, best, -1))
    logical = torch.where(there, best, 0)
    ids = tables[:, None].expand(-1, hkv, -1).gather(2, logical)
    head = torch.arange(hkv, device=lens.device)[None, :, None]
    keys, values = (state[c][ids, head].float().flatten(2, 3) for c in ("k_cache", "v_cache"))
    token = (logical[..., None] * block + torch.arange(block, device=lens.device))
    visible = ((token < lens[:, None, None, None]) & there[..., None]).flatten(2)
    return {"out": _attend(state["q"], keys, values, visible), "blocks": state["blocks"]}


# ------------------------------------------------------------------- work --
def work(case):
    hq, hkv, d, rows, block = (case[x] for x in ("q_heads", "kv_heads", "head_dim", "batch", "block"))
    lens = _lengths(case, 0)
    packed = d * 17 // 32
    if case["kind"] == "append":
        # q read and written, k and v read, quantised and written; the same slots read back as 16-bit values
        n = rows * case["new"]
        return {"bytes": n * (4 * hq * d + 8 * hkv * d + 4 * hkv * packed), "flops": 3 * n * (hq + hkv) * d}
    if case["kind"] == "fp4":
        tokens = sum(lens)
        return {"bytes": tokens * hkv * 2 * packed + rows * hq * d * 4, "flops": tokens * hq * d * 4}
    if case["kind"] == "bounds":
        fresh = sum(n // block - max(0, n - case["new"]) // block for n in lens)
        return {"bytes": rows * 4 + fresh * hkv * d * (2 * block + 4), "flops": 2 * fresh * hkv * d * block}
    counts = [-(-n // block) for n in lens]
    scored = sum(n - case["sinks"] - case["recent"] for n in counts if n > case["select"])
    tokens = sum(min(n, case["select"] * block) for n in lens)
    return {"bytes": scored * hkv * d * 4 + tokens * hkv * d * 4 + rows * hq * d * 4 + rows * hkv * case["select"] * 4,
            "flops": scored * hkv * d * 4 + tokens * hq * d * 4}


# ------------------------------------------------------------------ exact --
def exact(case, seed):
    """Row by row from the definitions, in 64 bits."""
    state = prepare(case, seed)
    return {"append": _exact_append, "fp4": _exact_fp4, "bounds": _exact_bounds, "sparse": _exact_sparse}[case["kind"]](
        case, state)


def _exact_levels(x):
    """float64 [..., D] rounded to the 4-bit format: the nearest level, of two the one with the even code."""
    x = x.unflatten(-1, (-1, 32))
    most = x.abs().amax(dim=-1, keepdim=True)
    e = torch.frexp(most / 7).exponent.double()  # 2^(e-1) <= most / 7 < 2^e
    unit = torch.exp2(torch.where(most / 7 == torch.exp2(e - 1), e - 1, e).clamp(-125, 125))
    level = torch.tensor(_LEVELS, device=x.device, dtype=torch.float64)
    a = (x / unit).abs()
    low = (torch.searchsorted(level, a.contiguous(), right=True) - 1).clamp(0, 6)
    below, above = a - level[low], level[low + 1] - a
    near = torch.where((above < below) | ((above == below) & (low % 2 == 1)), low + 1, low)
    return torch.copysign(level[near] * unit, x).flatten(-2)


def _exact_append(case, state):
    half, at = case["rotary"] // 2, state["positions"].long()
    c, s = (plane[at].double()[:, None] for plane in state["cos_sin"])
    result = {}
    for name in ("q", "k"):
        x = state[name].double()
        y = x.clone()
        y[..., :half] = x[..., :half] * c - x[..., half : 2 * half] * s
        y[..., half : 2 * half] = x[..., half : 2 * half] * c + x[..., :half] * s
        result[name] = y
    return {"q": result["q"], "k": _exact_levels(result["k"]), "v": _exact_levels(state["v"].double())}


def _exact_row(query, keys, values):
    p = torch.softmax(torch.mm(query, keys.t().contiguous()) / math.sqrt(query.shape[1]), dim=1)
    return torch.mm(p, values)


def _exact_unpack(pool, ids, off, h, block, d, values):
    """Tokens (ids, off) of head h, from the bytes."""
    page = pool[ids, h].long()
    n = torch.arange(len(ids), device=page.device)[:, None]
    dims, off = torch.arange(d, device=page.device)[None], off[:, None]
    code_at, scale_at = off * (d // 2) + dims // 2, off * (d // 32) + dims // 32
    if values:
        part = d // 16
        code_at = off // 4 * (2 * d) + dims // part * (2 * part) + off % 4 * (part // 2) + dims % part // 2
        scale_at = off // 4 * (d // 8) + dims // 32 * 4 + off % 4
    code = (page[n, code_at] >> (4 * (dims % 2))) & 15
    byte = page[n, block * d // 2 + scale_at]
    value = torch.tensor(_LEVELS, device=page.device, dtype=torch.float64)[code % 8]
    return torch.where(code >= 8, -value, value) * torch.exp2(byte.double() - 127)


def _exact_fp4(case, state):
    block, hkv, d = case["block"], case["kv_heads"], case["head_dim"]
    group = case["q_heads"] // hkv
    outs = []
    for b, n in enumerate(state["lens"].tolist()):
        seen = torch.arange(n, device="cuda")
        ids, off = state["tables"][b].long()[seen // block], seen % block
        for h in range(hkv):
            keys = _exact_unpack(state["k_cache"], ids, off, h, block, d, False)
            values = _exact_unpack(state["v_cache"], ids, off, h, block, d, True)
            outs.append(_exact_row(state["q"][b, h * group : (h + 1) * group].double(), keys, values))
    return torch.cat(outs).view(state["q"].shape)


def _exact_bounds(case, state):
    bounds, block, new = state["bounds"].double(), case["block"], case["new"]
    for row, n in zip(state["tables"].tolist(), state["lens"].tolist()):
        for j in range(max(0, n - new) // block, n // block):
            tokens = state["k_cache"][row[j]].double().sort(dim=1).values  # [Hkv, block, D]
            bounds[row[j], :, 0], bounds[row[j], :, 1] = tokens[:, 0], tokens[:, -1]
    return bounds


def _exact_sparse(case, state):
    block, hkv, select = case["block"], case["kv_heads"], case["select"]
    group = case["q_heads"] // hkv
    blocks = torch.full((case["batch"], hkv, select), -1, dtype=torch.int32)
    outs = []
    for b, n in enumerate(state["lens"].tolist()):
        count = -(-n // block)
        table = state["tables"][b].long()
        for h in range(hkv):
            query = state["q"][b, h * group : (h + 1) * group].double()
            chosen = list(range(count))
            if count > select:
                low, high = state["bounds"][table[:count], h].double().unbind(1)
                score = sum(torch.maximum(x * low, x * high).sum(dim=1) for x in query).float().tolist()
                inner = sorted(range(case["sinks"], count - case["recent"]), key=lambda j: (-score[j], j))
                chosen = sorted([*range(case["sinks"]), *inner[: select - case["sinks"] - case["recent"]],
                                 *range(count - case["recent"], count)])
            blocks[b, h, : len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
            seen = (torch.tensor(chosen)[:, None] * block + torch.arange(block)).flatten()
            seen = seen[seen < n].cuda()
            keys, values = (state[c][table[seen // block], h, seen % block].double() for c in ("k_cache", "v_cache"))
            outs.append(_exact_row(query, keys, values))
    return {"out": torch.cat(outs).view(state["q"].shape), "blocks": blocks.cuda()}
