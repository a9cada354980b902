"""The 4-bit cache format and its operators, in plain 64-bit forms from the definitions (CPU)."""

import math

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def block_bytes(block, d):
    return block * d * 17 // 32


def quantise(x):
    """(codes [..., D] 0..15, scale bytes [..., D / 32]) of values [..., D]."""
    x = x.detach().cpu().double().unflatten(-1, (-1, 32))
    amax = x.abs().amax(dim=-1)
    odd = ~torch.isfinite(x).all(dim=-1)
    amax = torch.where(odd, 1.0, amax)
    e = torch.full_like(amax, -125.0)
    for step in range(-125, 125):  # the least e with amax <= 7 * 2^e, at most 125
        e = torch.where(amax > 7 * 2.0**step, step + 1.0, e)
    y = torch.where(odd[..., None], 0.0, x) / torch.exp2(e)[..., None]
    dist = (y.abs()[..., None] - LEVELS).abs()  # (exact: y is a 24-bit value over a power of two)
    best = dist.amin(dim=-1, keepdim=True)
    ties = dist == best
    even = torch.arange(8) % 2 == 0
    code = torch.where((ties & even).any(dim=-1), (ties & even).byte().argmax(dim=-1), ties.byte().argmax(dim=-1))
    code = code + 8 * torch.signbit(y).long()
    code = torch.where(odd[..., None], 0, code)
    return code.flatten(-2), torch.where(odd, 255, e.long() + 127)


def places(block, d, values):
    """(byte, shift) of every code [block, D] and byte of every scale [block, D / 32] in a block."""
    tok, dim, group = torch.arange(block)[:, None], torch.arange(d)[None], torch.arange(d // 32)[None]
    shift = (4 * (dim % 2)).expand(block, d)
    if not values:
        return tok * (d // 2) + dim // 2, shift, block * d // 2 + tok * (d // 32) + group
    part = d // 16
    code = ((tok // 4 * 16 + dim // part) * 4 + tok % 4) * (part // 2) + dim % part // 2
    return code, shift, block * d // 2 + (tok // 4 * (d // 32) + group) * 4 + tok % 4


def unpack(pool, block, d, values):
    """float64 [num_blocks, heads, block, D] of a pool's bytes."""
    pool = pool.detach().cpu().long()
    code_at, shift, scale_at = places(block, d, values)
    code = (pool[..., code_at] >> shift) & 15
    byte = pool[..., scale_at]
    value = LEVELS[code % 8] * torch.where(code >= 8, -1.0, 1.0)
    scale = torch.where(byte == 255, math.nan, torch.exp2(byte.double() - 127))
    return value * scale.repeat_interleave(32, dim=-1)


def store(pool, ids, offsets, x, block, values):
    """Quantises x [tokens, heads, D] into a CPU pool's slots, in place; slots outside it are left out."""
    d = x.shape[-1]
    codes, scales = quantise(x)
    code_at, _, scale_at = places(block, d, values)
    for t, (blk, off) in enumerate(zip(ids.tolist(), offsets.tolist())):
        if 0 <= blk < pool.shape[0] and 0 <= off < block:
            pool[blk, :, code_at[off, ::2]] = (codes[t, :, ::2] | (codes[t, :, 1::2] << 4)).to(torch.uint8)
            pool[blk, :, scale_at[off]] = scales[t].to(torch.uint8)


def rotate(x, cos, sin, rotary):
    """float32 split-half rotation, each product and sum rounded on its own; cos, sin [tokens, rotary / 2]."""
    half = rotary // 2
    x = x.detach().cpu().float()
    c, s = cos[:, None], sin[:, None]
    x1, x2 = x[..., :half], x[..., half:rotary]
    return torch.cat((x1 * c - x2 * s, x2 * c + x1 * s, x[..., rotary:]), dim=-1)


def random_pool(blocks, heads, block, d, seed, values, spread=3):
    """A CPU pool of any codes and of scale bytes around 127."""
    gen = torch.Generator().manual_seed(seed)
    pool = torch.randint(0, 256, (blocks, heads, block_bytes(block, d)), generator=gen, dtype=torch.uint8)
    scales = torch.randint(125 - spread, 126 + spread, (blocks, heads, block * d // 32), generator=gen)
    pool[..., block * d // 2 :] = scales.to(torch.uint8)
    return pool


def attend(q, k, v, table, lens, scale=None):
    """(out [B, Hq, D], sum p |v|, largest sum |q k| and sum (largest |q| of 32 dims) |k|) in float64, of unpacked caches
    [num_blocks, heads, block, D]; tokens in blocks outside the pool are not attended."""
    q, table = q.detach().cpu().double(), table.detach().cpu()
    num_blocks, hkv, block, d = k.shape
    group = q.shape[1] // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    most = split = 0.0
    for b in range(q.shape[0]):
        at = torch.arange(min(max(int(lens[b]), 0), table.shape[1] * block))
        ids = table[b, at // block].long()
        at = at[(ids >= 0) & (ids < num_blocks)]
        ids = table[b, at // block].long()
        if not len(at):
            continue
        for h in range(hkv):
            heads = slice(h * group, (h + 1) * group)
            keys, values, x = k[ids, h, at % block], v[ids, h, at % block], q[b, heads]
            p = torch.softmax(x @ keys.t() * scale, dim=1)
            out[b, heads], size[b, heads] = p @ values, p @ values.abs()
            largest = x.abs().unflatten(1, (-1, 32)).amax(dim=2).repeat_interleave(32, dim=1)
            most = max(most, float((x.abs() @ keys.abs().t()).nan_to_num(0).max()))
            split = max(split, float((largest @ keys.abs().t()).nan_to_num(0).max()))
    return out, size, most, split
