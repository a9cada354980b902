"""Plain 64-bit forms of the bounded-cache operators, row by row from their definitions (CPU)."""

import math

import torch


def attended(length, window=None, sinks=0):
    """Token indices that a row of ``length`` tokens attends."""
    return [t for t in range(length) if window is None or t < sinks or t >= length - window]


def token_major(cache, kv_layout):
    return cache.transpose(2, 3) if kv_layout == "dim_major" else cache


def attend(q, k, v, table, lens, window=None, sinks=0, scale=None, kv_layout="token_major"):
    """(out [B, Hq, D], weights [B, Hkv, tokens]) in float64; tokens in blocks outside the pool are not attended."""
    q, table = q.detach().cpu().double(), table.detach().cpu()
    k, v = (token_major(c.detach().cpu(), kv_layout) for c in (k, v))
    num_blocks, hkv, block, d = k.shape
    batch, hq = q.shape[:2]
    group = hq // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    weights = torch.zeros(batch, hkv, table.shape[1] * block, dtype=torch.float64)
    for b in range(batch):
        length = min(max(int(lens[b]), 0), table.shape[1] * block)
        seen = [t for t in attended(length, window, sinks) if 0 <= int(table[b, t // block]) < num_blocks]
        if not seen:
            continue
        at = torch.tensor(seen)
        ids, off = table[b, at // block].long(), at % block
        for h in range(hkv):
            keys, values = k[ids, h, off].double(), v[ids, h, off].double()
            p = torch.softmax(q[b, h * group:(h + 1) * group] @ keys.t() * scale, dim=1)
            out[b, h * group:(h + 1) * group] = p @ values
            weights[b, h, at] = p.sum(dim=0)
    return out, weights


def kept_tokens(score, length, keep, sinks, recent):
    if length <= keep:
        return list(range(length))

    def rank(t):
        x = float(score[t])
        return (1, 0.0, t) if math.isnan(x) else (0, -x, t)

    inner = sorted(range(sinks, length - recent), key=rank)[: keep - sinks - recent]
    return sorted([*range(sinks), *inner, *range(length - recent, length)])


def evict(k, v, table, lens, scores, keep, sinks=0, recent=0, kv_layout="token_major"):
    """(kept, new lens, scores, K, V) after the call, on the CPU; K and V in the given layout."""
    num_blocks, block = k.shape[0], token_major(k, kv_layout).shape[2]
    table = table.detach().cpu()
    caches = [k.detach().cpu().clone(), v.detach().cpu().clone()]
    old = [token_major(c.clone(), kv_layout) for c in caches]
    new = [token_major(c, kv_layout) for c in caches]
    scores = scores.detach().cpu()
    new_scores = scores.clone()
    batch, hkv = scores.shape[:2]
    kept = torch.full((batch, hkv, keep), -1, dtype=torch.int32)
    new_lens = []
    for b in range(batch):
        length = min(max(int(lens[b]), 0), table.shape[1] * block)
        new_lens.append(min(length, keep))
        for h in range(hkv):
            stay = kept_tokens(scores[b, h], length, keep, sinks, recent)
            kept[b, h, : len(stay)] = torch.tensor(stay, dtype=torch.int32)
            new_scores[b, h, : len(stay)] = scores[b, h, stay] if stay else 0.0
            new_scores[b, h, len(stay):length] = 0.0
            for j, t in enumerate(stay):
                a, z = int(table[b, t // block]), int(table[b, j // block])
                if j != t and 0 <= a < num_blocks and 0 <= z < num_blocks:
                    for src, dst in zip(old, new):
                        dst[z, h, j % block] = src[a, h, t % block]
    return kept, torch.tensor(new_lens), new_scores, caches[0], caches[1]
