"""GPU parity of key bounds, block selection and attention over chosen blocks against their plain 64-bit forms
(tests/sparse_oracle.py).

Bounds and selections are compared exactly: bounds are values of the cache, and a score is a sum of at most 128 pairs of
products in 64 bits, rounded once to 32.  The sums that two orders give differ by at most 2^-45 of the terms' magnitudes, so
they round to different 32-bit numbers only next to a border between two of them, at odds of about 2^-20 a score, and that
matters only where the score is itself at the border of the selection.  The attention is the plain decode's, with the bound of
tests/test_bounded_gpu.py: |error| <= (u + 2 d + 2^-13) sum p |v| + u |out| and d <= (D + 2) 2^-24 scale log2(e) sum |q k|.
"""

import math
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

import flashdec_amd as fd
from flashdec_amd import paged_decode
from tests import fp4_oracle as fo
from tests import sparse_oracle as so
from tests.helpers import make_paged_inputs

pytestmark = pytest.mark.gpu

BF, HALF = torch.bfloat16, torch.float16
HALF_STEP = {BF: 2.0**-8, HALF: 2.0**-11}


def _inputs(lens, hq, hkv, d, block, dtype=BF, seed=1, kv_layout="token_major", index=torch.int32, width=None):
    q, k, v, table, lens = make_paged_inputs(lens, hq, hkv, d, block, dtype, seed, kv_layout=kv_layout, table_width=width)
    return 2 * q, k, v, table.to(index), lens.to(index)


def _bounds(k, table, lens, kv_layout="token_major"):
    shape = (k.shape[0], k.shape[1], 2, k.shape[3 if kv_layout == "token_major" else 2])
    return fd.paged_key_bounds(k, table, lens, torch.full(shape, 7.0, device="cuda", dtype=k.dtype), kv_layout=kv_layout)


def _same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0, 1, -1), b.nan_to_num(0, 1, -1)) and \
        torch.equal(a.isinf(), b.isinf())


def _check_attention(out, q, k, v, table, lens, blocks, scale=None, kv_layout="token_major"):
    want, size, most = so.attend(q, k, v, table, lens, blocks.cpu(), scale, kv_layout)
    d = q.shape[2]
    factor = math.log2(math.e) * (1.0 / math.sqrt(d) if scale is None else abs(scale))
    u, off = HALF_STEP[q.dtype], (d + 2) * 2.0**-24 * factor * most
    bound = (u + 2 * off + 2.0**-13) * size + u * want.abs() + 2.0**-24
    assert float(((out.cpu().double() - want).abs() - bound).max()) <= 0


@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("kv_layout", ["token_major", "dim_major"])
@pytest.mark.parametrize("hkv, d, block", [(2, 128, 32), (3, 64, 8), (8, 128, 16), (1, 64, 32)])
@pytest.mark.parametrize("new", [None, 0, 1, 7, 33, 100])
def test_bounds(dtype, kv_layout, hkv, d, block, new):
    _, k, _, table, lens = _inputs([700, 3, 0, 129, 2000, 64, 31, 1, 33, 32, 95, 512], hkv, hkv, d, block, dtype,
                                   kv_layout=kv_layout)
    k[5, 0, 1, 2], k[7, hkv - 1, 3, 0], k[9, 0, 0, 5] = math.nan, math.inf, -math.inf
    before = torch.full((k.shape[0], hkv, 2, d), 7.0, dtype=dtype)
    got = fd.paged_key_bounds(k, table, lens, before.cuda(), new_tokens=new, kv_layout=kv_layout)
    assert _same(got.cpu(), so.key_bounds(k, table, lens, before, new, kv_layout))


def test_bounds_of_odd_rows_and_views():
    _, k, _, table, lens = _inputs([200, 200, 90, 64], 2, 2, 128, 16, index=torch.int64, width=20)
    table[0, 2], table[1, 1], lens[2], lens[3] = -1, 10**6, -4, 10**6
    both = torch.stack((k, k + 1), dim=1)
    nhd = k.transpose(1, 2).contiguous().transpose(1, 2)  # tokens ahead of heads
    off = torch.zeros(k.numel() + 1, device="cuda", dtype=k.dtype)[1:].view(k.shape).copy_(k)
    before = torch.full((k.shape[0], 2, 2, 128), 7.0, dtype=k.dtype)
    want = so.key_bounds(k, table, lens, before)
    for cache in (k, both[:, 0], nhd, off):
        assert torch.equal(fd.paged_key_bounds(cache, table, lens, before.cuda()).cpu(), want)
    assert torch.equal(_bounds(k, table[:, ::2], lens).cpu(), so.key_bounds(k, table[:, ::2], lens, before))


def test_bounds_step_by_step_are_those_of_the_whole():
    _, k, _, table, lens = _inputs([200, 77, 32], 2, 2, 64, 8)
    grown = torch.zeros((k.shape[0], 2, 2, 64), device="cuda", dtype=k.dtype)
    whole = torch.zeros_like(grown)
    at = torch.zeros_like(lens)
    for step in (1, 30, 5, 64, 1, 1, 99):
        new = torch.minimum(at + step, lens)
        fd.paged_key_bounds(k, table, new, grown, new_tokens=step)
        at = new
    fd.paged_key_bounds(k, table, at, whole)
    assert torch.equal(grown, whole)


SELECTIONS = [(16, 1, 1), (5, 2, 3), (1, 0, 1), (40, 0, 2), (300, 1, 4)]


@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("hq, hkv, d, block, index", [(16, 2, 128, 32, torch.int32), (14, 2, 64, 8, torch.int64),
                                                      (8, 8, 128, 16, torch.int32), (71, 1, 64, 16, torch.int32)])
@pytest.mark.parametrize("n, sinks, recent", SELECTIONS)
def test_selection_and_attention(dtype, hq, hkv, d, block, index, n, sinks, recent):
    q, k, v, table, lens = _inputs([700, 3, 0, 129, 4000, 64, 31, 1, 33, 32, 95, 511], hq, hkv, d, block, dtype, index=index)
    bounds = _bounds(k, table, lens)
    chosen = fd.paged_block_select(q, k, bounds, table, lens, n, sinks, recent)
    want = so.select(q, bounds, table, lens, block, n, sinks, recent, hkv)
    for got, expect in zip(chosen, want):
        assert torch.equal(got.cpu(), expect)
    out = fd.paged_decode_attention_blocks(q, k, v, chosen, ragged=True)
    _check_attention(out, q, k, v, table, lens, chosen.blocks)


@pytest.mark.parametrize("length, block, n", [(70000, 8, 500), (40000, 32, 64), (131072, 16, 4096), (9000, 8, 1124)])
def test_long_rows(length, block, n):
    q, k, v, table, lens = _inputs([length, length // 3], 8, 2, 64, block)
    bounds = _bounds(k, table, lens)
    chosen = fd.paged_block_select(q, k, bounds, table, lens, n, 1, 2)
    for got, expect in zip(chosen, so.select(q, bounds, table, lens, block, n, 1, 2, 2)):
        assert torch.equal(got.cpu(), expect)
    _check_attention(fd.paged_decode_attention_blocks(q, k, v, chosen), q, k, v, table, lens, chosen.blocks)


def test_all_blocks_are_the_plain_decode():
    q, k, v, table, lens = _inputs([700, 3, 0, 129], 16, 2, 128, 32)
    chosen = fd.paged_block_select(q, k, _bounds(k, table, lens), table, lens, 64)
    out = fd.paged_decode_attention_blocks(q, k, v, chosen)
    _check_attention(out, q, k, v, table, lens, chosen.blocks)
    plain = fd.paged_decode_attention(q, k, v, table, lens)
    assert torch.allclose(out.float(), plain.float(), atol=2e-2, rtol=1e-2)


def test_ties_take_the_lowest_blocks():
    q, k, v, table, lens = _inputs([1000], 4, 2, 64, 8)
    bounds = torch.zeros((k.shape[0], 2, 2, 64), device="cuda", dtype=BF)
    table = table.long()
    bounds[table[0, 30:90], 0] = 1.0   # equal scores for a stretch
    bounds[table[0, 50], 1, 0] = -0.0  # equal to the zeros
    q[:] = q.abs()
    for n in (2, 3, 40, 62, 63, 100):
        got = fd.paged_block_select(q, k, bounds, table, lens, n, 0, 1)
        for g, w in zip(got, so.select(q, bounds, table, lens, 8, n, 0, 1, 2)):
            assert torch.equal(g.cpu(), w)
    chosen = fd.paged_block_select(q, k, bounds, table, lens, 40, 0, 1).blocks[0].tolist()
    assert chosen[0] == [*range(30, 69), 124] and chosen[1] == [*range(39), 124]


def test_scores_of_odd_values_and_blocks_outside_the_pool():
    q, k, v, table, lens = _inputs([1500, 900], 8, 2, 64, 16)
    bounds = _bounds(k, table, lens)
    table = table.long()
    bounds[table[0, 7], 0, 1, 3] = math.nan
    bounds[table[0, 60], 0, 0, 9] = math.nan
    bounds[table[0, 20], 1] = torch.tensor([-math.inf, math.inf], device="cuda")[:, None].expand(2, 64).to(BF)
    bounds[table[0, 21], 1] = torch.finfo(BF).max
    table[0, 9], table[0, 33], table[1, 5] = -1, k.shape[0], 2**31 - 1
    q[1, 0, 5] = math.nan  # every score of the head's rows: the first blocks
    for n in (3, 10, 50, 90):
        got = fd.paged_block_select(q, k, bounds, table, lens, n, 1, 1)
        for g, w in zip(got, so.select(q, bounds, table, lens, 16, n, 1, 1, 2)):
            assert torch.equal(g.cpu(), w)
    first = fd.paged_block_select(q, k, bounds, table, lens, 4, 1, 1).blocks.cpu()
    assert first[0, 0].tolist() == [0, 7, 60, 93] and first[1, 0].tolist() == [0, 1, 2, 56]
    out = fd.paged_decode_attention_blocks(q[:1], k, v, fd.paged_block_select(q[:1], k, bounds, table[:1], lens[:1], 60, 10, 1))
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("kv_layout", ["token_major", "dim_major"])
@pytest.mark.parametrize("hkv", [1, 3])
def test_layouts(kv_layout, hkv):
    q, k, v, table, lens = _inputs([700, 3, 0, 129], 2 * hkv, hkv, 128, 16, kv_layout=kv_layout)
    bounds = _bounds(k, table, lens, kv_layout)
    caches = [(k, v, hkv)]
    if kv_layout == "token_major":
        both = torch.stack((k, v), dim=1)
        nhd = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in (k, v)]
        caches += [(both[:, 0], both[:, 1], 2 * hkv if hkv > 1 else 1), (*nhd, 16 * hkv if hkv > 1 else 1)]
    for k2, v2, step in caches:
        chosen = fd.paged_block_select(q, k2, bounds, table, lens, 9, 1, 2, kv_layout=kv_layout)
        assert chosen.block_step == step
        for g, w in zip(chosen, so.select(q, bounds, table, lens, 16, 9, 1, 2, step)):
            assert torch.equal(g.cpu(), w)
        out = fd.paged_decode_attention_blocks(q, k2, v2, chosen, kv_layout=kv_layout)
        _check_attention(out, q, k, v, table, lens, chosen.blocks, kv_layout=kv_layout)


def test_strided_queries_and_outputs():
    q, k, v, table, lens = _inputs([700, 400], 8, 2, 128, 16)
    bounds = _bounds(k, table, lens)
    want = fd.paged_block_select(q, k, bounds, table, lens, 9, 1, 2)
    wide = torch.zeros(2, 8, 256, device="cuda", dtype=BF)[..., ::2]
    wide.copy_(q)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    for view in (wide, turned):
        got = fd.paged_block_select(view, k, bounds, table, lens, 9, 1, 2)
        assert all(torch.equal(g, w) for g, w in zip(got[:3], want[:3]))
        for out in (torch.empty_like(q), torch.empty(8, 2, 128, device="cuda", dtype=BF).transpose(0, 1),
                    torch.empty(2, 8, 256, device="cuda", dtype=BF)[..., ::2]):
            assert fd.paged_decode_attention_blocks_into(view, k, v, got, out) is out
            # (the plain decode of queries without unit dim stride is another kernel: equal within the bound)
            _check_attention(out, q, k, v, table, lens, got.blocks)


def _fp4_inputs(lens, hq, hkv, d, block, dtype, seed=1, index=torch.int32):
    q, _, _, table, lens = _inputs(lens, hq, hkv, d, block, dtype, seed, index=index)
    blocks = int(table.max()) + 3
    return q, *(fo.random_pool(blocks, hkv, block, d, seed + i, bool(i)).cuda() for i in range(2)), table, lens


def _check_4_bit_attention(out, q, keys, values, table, lens, blocks):
    d = q.shape[2]
    want, size, most = so.attend(q, keys, values, table, lens, blocks.cpu())
    largest = q.abs().unflatten(2, (-1, 32)).amax(dim=3).repeat_interleave(32, dim=2)
    split = so.attend(largest, keys, values, table, lens, blocks.cpu())[2]
    u = HALF_STEP[q.dtype]
    off = math.log2(math.e) / math.sqrt(d) * ((d + 2) * 2.0**-24 * most + 2.0**-21 * split)  # (as the 4-bit decode's tests)
    bound = (u + 2 * off + 2.0**-13) * size + u * want.abs() + 2.0**-24
    assert float(((out.cpu().double() - want).abs() - bound).max()) <= 0


@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("hkv, d, block", [(2, 128, 32), (3, 64, 8), (8, 128, 16), (1, 64, 32), (5, 128, 8)])
@pytest.mark.parametrize("new", [None, 1, 33])
def test_bounds_of_a_4_bit_cache(dtype, hkv, d, block, new):
    _, k, _, table, lens = _fp4_inputs([700, 3, 0, 129, 64, 31, 512], hkv, hkv, d, block, dtype)
    scale_at = fo.places(block, d, False)[2]
    k[table[0, 2].long(), 0, scale_at[5, 1]] = 255
    k[table[3, 1].long(), hkv - 1, scale_at[0, 0]] = 3  # (far below fp16's numbers)
    before = torch.full((k.shape[0], hkv, 2, d), 7.0, dtype=dtype)
    got = fd.paged_key_bounds(k, table, lens, before.cuda(), new_tokens=new)
    assert _same(got.cpu(), so.key_bounds(fo.unpack(k, block, d, False), table, lens, before, new))


@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("hq, hkv, d, block, index", [(16, 2, 128, 32, torch.int32), (14, 2, 64, 8, torch.int64),
                                                      (71, 1, 64, 16, torch.int32)])
@pytest.mark.parametrize("n, sinks, recent", [(16, 1, 1), (5, 2, 3), (300, 1, 4)])
def test_selection_and_attention_of_a_4_bit_cache(dtype, hq, hkv, d, block, index, n, sinks, recent):
    q, k, v, table, lens = _fp4_inputs([700, 3, 0, 129, 2000, 64, 33], hq, hkv, d, block, dtype, index=index)
    bounds = fd.paged_key_bounds(k, table, lens, torch.zeros((k.shape[0], hkv, 2, d), device="cuda", dtype=dtype))
    chosen = fd.paged_block_select(q, k, bounds, table, lens, n, sinks, recent)
    for got, expect in zip(chosen, so.select(q, bounds, table, lens, block, n, sinks, recent, hkv)):
        assert torch.equal(got.cpu(), expect)
    keys, values = fo.unpack(k, block, d, False), fo.unpack(v, block, d, True)
    both = torch.stack((k, v), dim=1)
    step = 2 * hkv if hkv > 1 else 1
    beside = fd.paged_block_select(q, both[:, 0], bounds, table, lens, n, sinks, recent)
    assert beside.block_step == step
    strided = torch.empty(hq, len(lens), d, device="cuda", dtype=dtype).transpose(0, 1)
    for out in (fd.paged_decode_attention_blocks(q, k, v, chosen),
                fd.paged_decode_attention_blocks(q, both[:, 0], both[:, 1], beside, kv_reuse=True),
                fd.paged_decode_attention_blocks(q, k, v, chosen, ragged=True),
                fd.paged_decode_attention_blocks_into(q, k, v, chosen, strided, sm_scale=d**-0.5, block_size=block)):
        _check_4_bit_attention(out, q, keys, values, table, lens, chosen.blocks)


def test_refusals_of_a_4_bit_cache():
    q, k, v, table, lens = _fp4_inputs([400, 90], 4, 2, 64, 16, BF)
    bounds = fd.paged_key_bounds(k, table, lens, torch.zeros((k.shape[0], 2, 2, 64), device="cuda", dtype=BF))
    chosen = fd.paged_block_select(q, k, bounds, table, lens, 4)
    wide = torch.zeros(*k.shape[:2], 2 * k.shape[2], device="cuda", dtype=torch.uint8)
    for call in (lambda: fd.paged_key_bounds(k, table, lens, bounds.float()),
                 lambda: fd.paged_key_bounds(k, table, lens, bounds[..., :32]),
                 lambda: fd.paged_key_bounds(k, table, lens, bounds[1:]),
                 lambda: fd.paged_key_bounds(k[..., :-16], table, lens, bounds),
                 lambda: fd.paged_key_bounds(wide[..., ::2], table, lens, bounds),
                 lambda: fd.paged_key_bounds(k, table, lens[:1], bounds),
                 lambda: fd.paged_key_bounds(k, table, lens, bounds, kv_layout="dim_major"),
                 lambda: fd.paged_key_bounds(k, table, lens, bounds, block_size=8),
                 lambda: fd.paged_block_select(q.half(), k, bounds, table, lens, 4),
                 lambda: fd.paged_block_select(q[:, :3], k, bounds, table, lens, 4),
                 lambda: fd.paged_block_select(q[..., :32], k, bounds, table, lens, 4),
                 lambda: fd.paged_block_select(q.float(), k, bounds, table, lens, 4),
                 lambda: fd.paged_block_select(q, k, bounds, table, lens, 4, kv_layout="dim_major"),
                 lambda: fd.paged_decode_attention_blocks(q, k, v, chosen, kv_layout="dim_major"),
                 lambda: fd.paged_decode_attention_blocks(q, k, v, chosen, block_size=8),
                 lambda: fd.paged_decode_attention_blocks(q, k, v[:, :1], chosen),
                 lambda: fd.paged_decode_attention_blocks(q.float(), k, v, chosen),
                 lambda: fd.paged_decode_attention_blocks(q, k, v.bfloat16(), chosen)):
        with pytest.raises(ValueError):
            call()


def test_captured_calls_and_streams():
    calls = [_inputs(lens, 8, 2, d, 16, seed=s) for lens, d, s in (([3000, 40], 128, 3), ([900] * 9, 64, 4))]
    bounds = [_bounds(k, table, lens) for _, k, _, table, lens in calls]
    outs = [torch.zeros_like(c[0]) for c in calls]

    def step(i, out):
        q, k, v, table, lens = calls[i]
        fd.paged_key_bounds(k, table, lens, bounds[i], new_tokens=1)
        return fd.paged_decode_attention_blocks_into(q, k, v, fd.paged_block_select(q, k, bounds[i], table, lens, 12, 1, 2), out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            step(i, outs[i])
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            step(i, outs[i])
    for turn in range(4):
        for (q, _, _, _, lens), out in zip(calls, outs):
            q.normal_()
            out.zero_()
            lens.sub_(turn)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], step(i, torch.empty_like(outs[i])))


def test_refusals():
    q, k, v, table, lens = _inputs([400, 90], 4, 2, 64, 16)
    bounds = _bounds(k, table, lens)
    sel = fd.paged_block_select
    for args, message in (
            ((q, k, bounds, table, lens, 0), "num_select"), ((q, k, bounds, table, lens, True), "num_select"),
            ((q, k, bounds, table, lens, 4, 2, 3), "must hold"), ((q, k, bounds, table, lens, 4, 1, 0), "recent_blocks"),
            ((q, k, bounds, table, lens, 4, -1, 1), "sink_blocks"), ((q, k, bounds[1:], table, lens, 4), "bounds must have shape"),
            ((q, k, bounds.half(), table, lens, 4), "cache's dtype"), ((q, k, bounds.cpu(), table, lens, 4), "device"),
            ((q, k, bounds.transpose(2, 3).contiguous().transpose(2, 3), table, lens, 4), "contiguous"),
            ((q[:, :3], k, bounds, table, lens, 4), "divisible"), ((q[:1], k, bounds, table, lens, 4), "one row/value"),
            ((q.cpu(), k, bounds, table, lens, 4), "CUDA"), ((q, k, bounds, table.float(), lens, 4), "int32 or int64"),
            ((q, k[:, :1].expand(-1, 2, -1, -1), bounds, table, lens, 4), "block stride")):
        with pytest.raises(ValueError, match=message):
            sel(*args)
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        sel(None, k, bounds, table, lens, 4)
    odd = torch.zeros(bounds.numel() + 1, device="cuda", dtype=BF)[1:].view_as(bounds)
    sel(q, k, bounds, table, lens, 4)
    for call in (lambda: sel(q, k, odd, table, lens, 4), lambda: fd.paged_key_bounds(k, table, lens, odd)):
        with pytest.raises(ValueError, match="16-byte line"):
            call()
    for bad in (-1, True, 1.5):
        with pytest.raises(ValueError, match="new_tokens"):
            fd.paged_key_bounds(k, table, lens, bounds, new_tokens=bad)
    blocks, tables, ln = (torch.empty(s, device="cuda", dtype=torch.int32) for s in ((2, 2, 4), (2, 2, 4), (2, 2)))
    for outs, message in (((blocks.long(), tables, ln), "int32"), ((blocks[:1], tables, ln), "shape"),
                          ((blocks, tables[..., :3], ln), "shape of blocks"), ((blocks, tables, ln[:1]), "shape of blocks"),
                          ((blocks, tables.transpose(0, 1), ln), "contiguous"), ((blocks, blocks, ln), "different tensors")):
        with pytest.raises(ValueError, match=message):
            fd.paged_block_select_into(q, k, bounds, table, lens, *outs)
    chosen = sel(q, k, bounds, table, lens, 4)
    with pytest.raises(TypeError, match="BlockSelection"):
        fd.paged_decode_attention_blocks(q, k, v, chosen.blocks)
    nhd = k.transpose(1, 2).contiguous().transpose(1, 2)
    for args in ((q, nhd, v, chosen), (q, k, nhd, chosen), (q[:1], k, v, chosen), (q, k[:, :1], v[:, :1], chosen),
                 (q[:, :3], k, v, chosen)):
        with pytest.raises(ValueError):
            fd.paged_decode_attention_blocks(*args)


def test_caches_past_four_gigabytes():
    q, k, v, table, lens = _inputs([900, 70], 8, 2, 128, 32)
    far = (1 << 32) // (2 * k[0].numel()) + 5
    pools = [torch.empty((far + k.shape[0], *k.shape[1:]), device="cuda", dtype=BF) for _ in range(2)]
    for pool, small in zip(pools, (k, v)):
        pool[far:] = small
    bounds, near = (torch.zeros((n, 2, 2, 128), device="cuda", dtype=BF) for n in (pools[0].shape[0], k.shape[0]))
    moved = torch.where(table < 0, table, table + far)
    fd.paged_key_bounds(pools[0], moved, lens, bounds)
    fd.paged_key_bounds(k, table, lens, near)
    assert torch.equal(bounds[far:], near)
    chosen = fd.paged_block_select(q, pools[0], bounds, moved, lens, 9, 1, 2)
    want = fd.paged_block_select(q, k, near, table, lens, 9, 1, 2)
    assert torch.equal(chosen.blocks, want.blocks) and torch.equal(chosen.lens, want.lens)
    assert torch.equal(fd.paged_decode_attention_blocks(q, *pools, chosen), fd.paged_decode_attention_blocks(q, k, v, want))


@pytest.mark.parametrize("dtype, hq, hkv, d, block", [(BF, 16, 2, 128, 16), (HALF, 6, 3, 64, 8)])
@pytest.mark.parametrize("fp4", [False, True])
def test_prompts_and_steps(dtype, hq, hkv, d, block, fp4):
    """Two prompts and a dozen steps: append, bounds of what it completed, selection, attention over it."""
    gen = torch.Generator().manual_seed(5)
    shape = (40, hkv, fd.fp4_block_bytes(block, d)) if fp4 else (40, hkv, block, d)
    k_cache, v_cache = (torch.zeros(shape, dtype=torch.uint8 if fp4 else dtype, device="cuda") for _ in range(2))
    append = fd.fused_rope_kv_append_fp4 if fp4 else fd.fused_rope_kv_append
    bounds = torch.zeros(40, hkv, 2, d, dtype=dtype, device="cuda")
    table = torch.randperm(40, generator=gen).view(2, 20).cuda()
    lens = torch.zeros(2, dtype=torch.int64, device="cuda")
    n, sinks, recent = 4, 1, 1
    for step in range(13):
        new = (100, 61) if step == 0 else (1, 1)
        at = torch.cat([int(x) + torch.arange(m) for x, m in zip(lens, new)]).cuda()
        row = torch.repeat_interleave(torch.arange(2), torch.tensor(new)).cuda()
        q, k, v = (torch.randn(len(at), h, d, generator=gen).to(dtype).cuda() for h in (hq, hkv, hkv))
        rotated = append(2 * q, k, v, k_cache, v_cache, table[row, at // block], at % block, at)
        lens += torch.tensor(new).cuda()
        last = rotated[lens.cumsum(0) - 1] if step == 0 else rotated
        fd.paged_key_bounds(k_cache, table, lens, bounds, new_tokens=None if step == 0 else 1)
        keys, values = (fo.unpack(k_cache, block, d, False), fo.unpack(v_cache, block, d, True)) if fp4 else (k_cache, v_cache)
        whole = so.key_bounds(keys, table, lens, torch.zeros_like(bounds))
        assert torch.equal(bounds.cpu(), whole)
        chosen = fd.paged_block_select(last, k_cache, bounds, table, lens, n, sinks, recent)
        for got, expect in zip(chosen, so.select(last, whole, table, lens, block, n, sinks, recent, hkv)):
            assert torch.equal(got.cpu(), expect)
        out = fd.paged_decode_attention_blocks(last, k_cache, v_cache, chosen)
        if fp4:
            _check_4_bit_attention(out, last, keys, values, table, lens, chosen.blocks)
        else:
            _check_attention(out, last, keys, values, table, lens, chosen.blocks)


def test_threads_on_one_stream():
    """Calls of several threads at once: each has its own keys and partials."""
    jobs = [_inputs(lens, 8, 2, d, 16, seed=s) for lens, d, s in (([3000, 40], 128, 3), ([900] * 9, 64, 4), ([5000], 64, 5))]
    bounds = [_bounds(k, table, lens) for _, k, _, table, lens in jobs]

    def run(i):
        q, k, v, table, lens = jobs[i]
        return fd.paged_decode_attention_blocks(q, k, v, fd.paged_block_select(q, k, bounds[i], table, lens, 12, 1, 2))

    want = [run(i) for i in range(3)]
    torch.cuda.synchronize()
    with ThreadPoolExecutor(3) as pool:
        got = [[f.result(timeout=60) for f in [pool.submit(run, i) for i in range(3)]] for _ in range(20)]
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("length, block", [(1500, 16), (3000, 8), (9000, 8), (40000, 8)])
@pytest.mark.parametrize("n, sinks, recent", [(2, 1, 1), (1, 0, 1), (5, 0, 5), (7, 4, 3)])
def test_sinks_and_recent_blocks_that_fill_the_list(length, block, n, sinks, recent):
    """No place is left for a scored block, whatever the scores are: of bounds that were never written, or of a NaN query."""
    q, k, v, table, lens = _inputs([length, length // 3, 20], 8, 2, 64, block)
    bounds = torch.full((k.shape[0], 2, 2, 64), math.nan, device="cuda", dtype=BF)
    chosen = fd.paged_block_select(q, k, bounds, table, lens, n, sinks, recent)
    for g, w in zip(chosen, so.select(q, bounds, table, lens, block, n, sinks, recent, 2)):
        assert torch.equal(g.cpu(), w)
    _check_attention(fd.paged_decode_attention_blocks(q, k, v, chosen), q, k, v, table, lens, chosen.blocks)
    bounds = _bounds(k, table, lens)
    bounds[table[0, length // block // 2].long(), 0, 1, 3] = math.nan
    q[1, 0, 5] = math.nan
    for g, w in zip(fd.paged_block_select(q, k, bounds, table, lens, n, sinks, recent),
                    so.select(q, bounds, table, lens, block, n, sinks, recent, 2)):
        assert torch.equal(g.cpu(), w)


FAR = (2**32, -(2**32), 5 * 2**32)  # added to a 64-bit id, these leave its low word as it is


@pytest.mark.parametrize("kv_layout", ["token_major", "dim_major"])
def test_bounds_leave_out_ids_past_32_bits(kv_layout):
    _, k, _, table, lens = _inputs([200, 90, 64], 2, 2, 128, 16, index=torch.int64, kv_layout=kv_layout)
    for b, j, far in zip((0, 0, 1), (2, 7, 1), FAR):
        table[b, j] += far
    before = torch.full((k.shape[0], 2, 2, 128), 7.0, dtype=k.dtype)
    got = fd.paged_key_bounds(k, table, lens, before.cuda(), kv_layout=kv_layout).cpu()
    assert torch.equal(got, so.key_bounds(k, table, lens, before, None, kv_layout))
    _, k, _, table, lens = _fp4_inputs([200, 90, 64], 2, 2, 128, 16, BF, index=torch.int64)
    for b, j, far in zip((0, 0, 1), (2, 7, 1), FAR):
        table[b, j] += far
    before = torch.full((k.shape[0], 2, 2, 128), 7.0, dtype=BF)
    got = fd.paged_key_bounds(k, table, lens, before.cuda()).cpu()
    assert torch.equal(got, so.key_bounds(fo.unpack(k, 16, 128, False), table, lens, before))


@pytest.mark.parametrize("width", [None, 700])
def test_selection_ranks_ids_past_32_bits_last(width):
    q, k, v, table, lens = _inputs([1500, 900], 8, 2, 64, 16, index=torch.int64, width=width)
    bounds = _bounds(k, table, lens)
    for b, j, far in zip((0, 0, 1), (93, 40, 0), FAR):
        table[b, j] += far
    for n in (3, 50, 93, 94, 100):
        chosen = fd.paged_block_select(q, k, bounds, table, lens, n, 1, 1)
        for g, w in zip(chosen, so.select(q, bounds, table, lens, 16, n, 1, 1, 2)):
            assert torch.equal(g.cpu(), w)
        _check_attention(fd.paged_decode_attention_blocks(q, k, v, chosen), q, k, v, table, lens, chosen.blocks)


def test_outputs_of_the_selection_that_share_elements_are_refused():
    q, k, v, table, lens = _inputs([400, 90], 4, 2, 64, 16)
    bounds = _bounds(k, table, lens)
    flat = torch.zeros(64, device="cuda", dtype=torch.int32)

    def at(x):  # blocks and tables of 16 numbers each, lens of 4
        return [flat[a : a + n].view(2, 2, -1) for a, n in zip(x, (16, 16, 4))]

    for x in ((0, 15, 40), (15, 0, 40), (0, 16, 31), (0, 16, 15), (20, 40, 17), (20, 40, 37), (20, 40, 55)):
        blocks, tables, ln = at(x)
        for _ in range(2):
            with pytest.raises(ValueError, match="share no element"):
                fd.paged_block_select_into(q, k, bounds, table, lens, blocks, tables, ln.view(2, 2))
    assert not bool(flat.any())
    want = fd.paged_block_select(q, k, bounds, table, lens, 4)
    for x in ((0, 16, 32), (16, 0, 32), (20, 40, 16), (20, 40, 36), (20, 40, 56)):
        blocks, tables, ln = at(x)
        got = fd.paged_block_select_into(q, k, bounds, table, lens, blocks, tables, ln.view(2, 2))
        assert all(torch.equal(g, w) for g, w in zip(got[:3], want[:3]))


def test_an_output_with_overlapping_elements_is_refused():
    for q, k, v, table, lens in (_inputs([400, 90], 4, 2, 64, 16), _fp4_inputs([400, 90], 4, 2, 64, 16, BF)):
        bounds = torch.zeros((k.shape[0], 2, 2, 64), device="cuda", dtype=BF)
        chosen = fd.paged_block_select(q, k, bounds, table, lens, 4)
        for out in (q[:1].expand(2, 4, 64), q[:, :1].expand(2, 4, 64), torch.zeros(700, device="cuda", dtype=BF).as_strided(
                (2, 4, 64), (128, 32, 1))):
            with pytest.raises(ValueError, match="overlapping"):
                fd.paged_decode_attention_blocks_into(q, k, v, chosen, out)


def test_kept_calls_hold_no_split_workspace_that_a_larger_one_replaced():
    calls = []
    for n in (1, 2, 3, 4, 6):
        q, k, v, table, lens = _inputs([3000] * n, 16, 2, 128, 16, seed=n)
        chosen = fd.paged_block_select(q, k, _bounds(k, table, lens), table, lens, 100, 1, 2)
        calls.append((q, k, v, chosen, torch.zeros_like(q), table, lens))
    side = torch.cuda.Stream()  # (whose workspaces are new)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        before = torch.cuda.memory_allocated()
        for _ in range(2):
            for q, k, v, chosen, out, _, _ in calls:
                fd.paged_decode_attention_blocks_into(q, k, v, chosen, out)
        held = paged_decode._WORKSPACES.__dict__.pop((q.device.index, side.cuda_stream))
        grown = torch.cuda.memory_allocated() - before
        mine = held.flat.numel() * 4 + held.counters.numel() * 4
        assert grown <= mine + 4096  # (the allocator's steps)
        del held
        assert torch.cuda.memory_allocated() <= before + 4096
        for q, k, v, chosen, out, table, lens in calls:  # a new one
            _check_attention(fd.paged_decode_attention_blocks_into(q, k, v, chosen, out), q, k, v, table, lens, chosen.blocks)


def test_lists_that_hold_the_whole_table_allocate_nothing_but_their_outputs():
    q, k, v, table, lens = _inputs([9000, 4000], 8, 2, 64, 8)
    bounds = _bounds(k, table, lens)
    outs = [torch.empty(s, device="cuda", dtype=torch.int32) for s in ((2, 2, 1125), (2, 2, 1125), (2, 2))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        before = torch.cuda.memory_allocated()
        chosen = fd.paged_block_select_into(q, k, bounds, table, lens, *outs)
        assert torch.cuda.memory_allocated() == before
    torch.cuda.synchronize()
    for g, w in zip(chosen, so.select(q, bounds, table, lens, 8, 1125, 1, 1, 2)):
        assert torch.equal(g.cpu(), w)
