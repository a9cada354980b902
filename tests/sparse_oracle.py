"""Plain 64-bit forms of the block-selecting operators, row by row from their definitions (CPU)."""

import math

import numpy as np
import torch

from tests.bounded_oracle import token_major


def key_bounds(k, table, lens, bounds, new_tokens=None, kv_layout="token_major"):
    """``bounds`` after the call, on the CPU."""
    k, bounds = token_major(k.detach().cpu(), kv_layout), bounds.detach().cpu().clone()
    block = k.shape[2]
    for row, n in zip(table.tolist(), lens.tolist()):
        n = min(max(n, 0), len(row) * block)
        first = 0 if new_tokens is None else max(0, n - new_tokens) // block
        for j in range(first, n // block):
            if 0 <= row[j] < k.shape[0]:
                keys = k[row[j]].double()
                odd = keys.isnan().any(dim=1)
                for i, x in enumerate((keys.nan_to_num(math.inf, math.inf, -math.inf).amin(dim=1),
                                       keys.nan_to_num(-math.inf, math.inf, -math.inf).amax(dim=1))):
                    bounds[row[j], :, i] = torch.where(odd, math.nan, x).to(bounds.dtype)
    return bounds


def scores(q, bounds, ids):
    """32-bit scores of the blocks ``ids`` (a list of pool ids) for one KV head's queries [G, D]; bounds [num_blocks, 2, D]."""
    q = q.detach().cpu().double()
    up, down = q.clamp_min(0).sum(dim=0), q.clamp_max(0).sum(dim=0)
    low, high = bounds.detach().cpu()[torch.tensor(ids, dtype=torch.int64)].double().unbind(1)
    return (up * high + down * low).sum(dim=1).to(torch.float32)


def select(q, bounds, table, lens, block, n, sinks, recent, block_step):
    """(blocks, tables, lens) on the CPU."""
    num_blocks, hkv = bounds.shape[:2]
    group = q.shape[1] // hkv
    blocks = torch.full((len(lens), hkv, n), -1, dtype=torch.int32)
    tables, out_lens = blocks.clone(), torch.zeros(len(lens), hkv, dtype=torch.int32)
    for b, (row, length) in enumerate(zip(table.tolist(), lens.tolist())):
        length = min(max(length, 0), len(row) * block)
        count = -(-length // block)
        for h in range(hkv):
            chosen = list(range(count))
            if count > n:
                inner = [j for j in range(sinks, count - recent)]
                held = [j for j in inner if 0 <= row[j] < num_blocks]
                value = dict(zip(held, scores(q[b, h * group:(h + 1) * group], bounds[:, h], [row[j] for j in held]).tolist()))

                def rank(j):
                    x = value.get(j)
                    return (2, 0.0, j) if x is None else (0, 0.0, j) if math.isnan(x) else (1, -x, j)

                inner.sort(key=rank)
                chosen = sorted([*range(sinks), *inner[: n - sinks - recent], *range(count - recent, count)])
            blocks[b, h, : len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
            ids = [row[j] * block_step + h if 0 <= row[j] < num_blocks else -1 for j in chosen]
            tables[b, h, : len(ids)] = torch.from_numpy(np.array(ids, dtype=np.int32))
            out_lens[b, h] = sum(min(block, length - j * block) for j in chosen)
    return blocks, tables, out_lens


def attend(q, k, v, table, lens, blocks, scale=None, kv_layout="token_major"):
    """(out, sum p |v|, largest sum |q k|) over the chosen blocks, float64."""
    q = q.detach().cpu().double()
    k, v = (token_major(c.detach().cpu(), kv_layout).double() for c in (k, v))
    num_blocks, hkv, block, d = k.shape
    group = q.shape[1] // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out, size, most = torch.zeros_like(q), torch.zeros_like(q), 0.0
    for b, row in enumerate(table.tolist()):
        length = min(max(int(lens[b]), 0), len(row) * block)
        for h in range(hkv):
            seen = [t for j in blocks[b, h].tolist() if j >= 0 and 0 <= row[j] < num_blocks
                    for t in range(j * block, min(length, (j + 1) * block))]
            if not seen:
                continue
            at = torch.tensor(seen)
            ids = torch.tensor(row)[at // block].long()
            heads = slice(h * group, (h + 1) * group)
            keys, values = k[ids, h, at % block], v[ids, h, at % block]
            p = torch.softmax(q[b, heads] @ keys.t() * scale, dim=1)
            out[b, heads], size[b, heads] = p @ values, p @ values.abs()
            most = max(most, float((q[b, heads].abs() @ keys.abs().t()).max()))
    return out, size, most
