"""GPU parity of the 4-bit cache's append and read against their plain forms (tests/fp4_oracle.py): every byte and
every value exactly, as the format's rounding is of exactly known numbers (the rotation's products and sums are rounded
one by one, from the same cos/sin)."""

import math

import numpy as np
import pytest
import torch

import flashdec_amd as fd
from flashdec_amd import rope
from tests import fp4_oracle as fo

pytestmark = pytest.mark.gpu

BF, HALF = torch.bfloat16, torch.float16


def _pools(blocks, heads, block, d, fill=0xA5):
    return [torch.full((blocks, heads, fo.block_bytes(block, d)), fill, dtype=torch.uint8, device="cuda") for _ in range(2)]


def _tokens(n, hq, hkv, d, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    qkv = torch.randn(n, hq + 2 * hkv, d, generator=gen)
    qkv *= torch.exp2(torch.randint(-6, 5, (n, hq + 2 * hkv, 1), generator=gen).float())
    return qkv.to(dtype).cuda().split((hq, hkv, hkv), dim=1)


def _slots(n, blocks, block, seed, index=torch.int64):
    gen = torch.Generator().manual_seed(seed)
    at = torch.randperm(blocks * block, generator=gen)[:n]
    return (at // block).to(index).cuda(), (at % block).to(index).cuda()


def _table(rows, rotary):
    return rope.rope_cos_sin_table(rows, rotary)


def _check(q, k, v, pools, before, ids, offsets, block, q_out, cos_sin, positions, rotary):
    at = positions.cpu().long().clamp(0, cos_sin.shape[1] - 1)
    cos, sin = cos_sin.cpu()[:, at]
    assert torch.equal(q_out.cpu(), fo.rotate(q, cos, sin, rotary).to(q.dtype))
    for pool, old, x, values in zip(pools, before, (fo.rotate(k, cos, sin, rotary), v), (False, True)):
        want = old.clone()
        fo.store(want, ids.cpu(), offsets.cpu(), x, block, values)
        assert torch.equal(pool.cpu(), want)


@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("n, hq, hkv, d, block, rotary", [
    (1, 16, 2, 128, 16, 128), (5, 32, 8, 128, 32, 64), (37, 14, 2, 64, 8, 64), (200, 3, 3, 64, 16, 32),
    (9, 71, 1, 64, 32, 20), (33, 5, 5, 128, 8, 2), (600, 16, 2, 128, 32, 128), (3, 300, 20, 128, 16, 42),
    (2051, 2, 1, 64, 8, 64)])
def test_append_stores_the_format(dtype, n, hq, hkv, d, block, rotary):
    q, k, v = _tokens(n, hq, hkv, d, dtype, n)  # (slices of one projection: neither is contiguous)
    blocks = n // block + 3
    pools = _pools(blocks, hkv, block, d)
    before = [p.cpu() for p in pools]
    ids, offsets = _slots(n, blocks, block, n)
    positions = torch.randint(0, 500, (n,), generator=torch.Generator().manual_seed(n)).cuda()
    table = _table(500, rotary)
    q_out = fd.fused_rope_kv_append_fp4(q, k, v, *pools, ids, offsets, positions, rotary_dim=rotary, cos_sin_table=table)
    _check(q, k, v, pools, before, ids, offsets, block, q_out, table, positions, rotary)


@pytest.mark.parametrize("rotary", [128, 64, 36])
def test_append_without_a_table_rotates_as_the_16_bit_append(rotary):
    q, k, v = (x.contiguous() for x in _tokens(50, 8, 2, 128, BF, 4))
    pools, caches = _pools(6, 2, 16, 128), [torch.zeros(6, 2, 16, 128, dtype=torch.float32, device="cuda") for _ in range(2)]
    ids, offsets = _slots(50, 6, 16, 4)
    positions = torch.arange(50, device="cuda") * 977
    got = fd.fused_rope_kv_append_fp4(q, k, v, *pools, ids, offsets, positions, rotary_dim=rotary, base=5e5)
    # the 16-bit append on 32-bit tensors leaves the 32-bit rotation in its cache
    want = fd.fused_rope_kv_append(q.float(), k.float(), v.float(), *caches, ids, offsets, positions, rotary_dim=rotary,
                                   base=5e5)
    assert torch.equal(got, want.to(BF))
    rotated = caches[0][ids, :, offsets]
    expect = torch.full(pools[0].shape, 0xA5, dtype=torch.uint8)
    fo.store(expect, ids.cpu(), offsets.cpu(), rotated, 16, False)
    assert torch.equal(pools[0].cpu(), expect)


@pytest.mark.parametrize("d", [64, 128])
def test_append_without_rotation(d):
    _, k, v = _tokens(21, 1, 3, d, BF, 8)
    pools = _pools(4, 3, 8, d)
    before = [p.cpu() for p in pools]
    ids, offsets = _slots(21, 4, 8, 8, torch.int32)
    fd.kv_append_fp4(k, v, *pools, ids, offsets)
    for pool, old, x, values in zip(pools, before, (k, v), (False, True)):
        fo.store(old, ids.cpu(), offsets.cpu(), x, 8, values)
        assert torch.equal(pool.cpu(), old)


@pytest.mark.parametrize("dtype", [BF, HALF])
def test_groups_of_odd_values(dtype):
    """Zeros, ties, the type's ends, infinities and NaN: a group that holds one of the last two is NaN as a whole."""
    x = torch.randn(12, 2, 64, generator=torch.Generator().manual_seed(1))
    x[0] = 0.0
    x[1] = -0.0
    x[2, 0, 3], x[2, 1, 40], x[3, 0, 63], x[4, 1, 0] = math.nan, math.inf, -math.inf, -math.nan
    x[5] = torch.finfo(dtype).max
    x[6] = torch.finfo(dtype).tiny / 4  # below the normal numbers
    x[7, :, ::2], x[7, :, 1] = 0.0, torch.finfo(dtype).max
    ties = torch.tensor([7.0, 0.25, -0.75, 1.25, 1.75, -2.5, 3.5, 5.0]).repeat(8)
    x[8] = ties
    x[9], x[10], x[11] = ties * 2.0**-10, ties * 7 / 8, torch.linspace(-7, 7, 64)
    x = x.to(dtype).cuda()
    pools = _pools(2, 2, 8, 64)
    before = [p.cpu() for p in pools]
    ids, offsets = _slots(12, 2, 8, 2)
    fd.kv_append_fp4(x, x, *pools, ids, offsets)
    for pool, old, values in zip(pools, before, (False, True)):
        fo.store(old, ids.cpu(), offsets.cpu(), x, 8, values)
        assert torch.equal(pool.cpu(), old)
    for got, values in zip(fd.paged_kv_read_fp4(*pools, ids, offsets, 64), (False, True)):
        want = fo.unpack(pools[0 if not values else 1], 8, 64, values)[ids.cpu(), :, offsets.cpu()]
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want)) and int(torch.isnan(got).sum()) == 4 * 32
        assert torch.equal(got.cpu().double().nan_to_num(0), want.nan_to_num(0))


@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("block, d", [(8, 64), (16, 128), (32, 64), (32, 128)])
def test_read_gives_any_bytes(dtype, block, d):
    pools = []
    for values in (False, True):
        pool = fo.random_pool(5, 3, block, d, 7 + values, values)
        gen = torch.Generator().manual_seed(9)
        pool[1:, :, block * d // 2 :] = torch.randint(0, 256, pool[1:, :, block * d // 2 :].shape, generator=gen).to(torch.uint8)
        pools.append(pool.cuda())
    ids, offsets = (x.flatten() for x in torch.meshgrid(torch.arange(5), torch.arange(block), indexing="ij"))
    ids, offsets = torch.cat((ids, torch.tensor([-1, 5, 2, 2, 2**33]))), torch.cat((offsets, torch.tensor([0, 0, -1, block, 1])))
    k, v = fd.paged_kv_read_fp4(*pools, ids.cuda(), offsets.cuda(), d, dtype)
    n = 5 * block
    for got, pool, values in ((k, pools[0], False), (v, pools[1], True)):
        want = fo.unpack(pool, block, d, values)[ids[:n], :, offsets[:n]].float()
        want = torch.cat((want, torch.zeros(5, 3, d))).to(dtype)  # (a 32-bit float holds every value of the format)
        assert torch.equal(got.isnan().cpu(), want.isnan())
        assert torch.equal(got.cpu().nan_to_num(0, 1, -1), want.nan_to_num(0, 1, -1))
        assert torch.equal(got.isinf().cpu(), want.isinf())


@pytest.mark.parametrize("heads, d, n", [(8, 128, 4099), (8, 64, 8195), (20, 128, 1401), (1, 128, 33000)])
def test_reads_that_fill_the_card(heads, d, n):
    """Several groups of tokens a workgroup, the last ones not there: the values of smaller calls."""
    pools = [fo.random_pool(40, heads, 16, d, 3 + i, bool(i)).cuda() for i in range(2)]
    gen = torch.Generator().manual_seed(n)
    ids, offsets = torch.randint(-1, 41, (n,), generator=gen).cuda(), torch.randint(0, 16, (n,), generator=gen).int().cuda()
    whole = fd.paged_kv_read_fp4(*pools, ids, offsets, d)
    for at in range(0, n, 200):
        part = fd.paged_kv_read_fp4(*pools, ids[at : at + 200], offsets[at : at + 200], d)
        assert all(torch.equal(w[at : at + 200], p) for w, p in zip(whole, part))


def test_slots_outside_the_cache():
    q, k, v = _tokens(6, 4, 2, 128, BF, 3)
    pools = _pools(3, 2, 16, 128)
    before = [p.cpu() for p in pools]
    ids = torch.tensor([0, -1, 3, 1, 2**32 + 1, 2], device="cuda")
    offsets = torch.tensor([3, 3, 3, 16, 3, -1], device="cuda")
    positions = torch.arange(6, device="cuda")
    table = _table(4, 128)
    with pytest.raises(ValueError, match="block_ids must be within"):
        fd.fused_rope_kv_append_fp4(q, k, v, *pools, ids, offsets, positions)
    with pytest.raises(ValueError, match="block_offsets must be within"):
        fd.kv_append_fp4(k, v, *pools, ids.clamp(0, 2), offsets)
    with pytest.raises(ValueError, match="positions must be non-negative"):
        fd.fused_rope_kv_append_fp4(q, k, v, *pools, ids.clamp(0, 2), offsets.clamp(0, 15), positions - 1)
    with pytest.raises(ValueError, match="below the cos_sin_table's rows"):
        fd.fused_rope_kv_append_fp4(q, k, v, *pools, ids.clamp(0, 2), offsets.clamp(0, 15), positions, cos_sin_table=table)
    for pool, old in zip(pools, before):
        assert torch.equal(pool.cpu(), old)
    q_out = fd.fused_rope_kv_append_fp4(q, k, v, *pools, ids, offsets, positions, cos_sin_table=table, check_indices=False)
    _check(q, k, v, pools, before, ids, offsets, 16, q_out, table, positions, 128)  # (only the first token is stored)


def test_tensors_off_the_16_byte_lines_and_pools_of_any_strides():
    qkv = torch.randn(7, 20, 133, device="cuda").to(HALF)
    q, k, v = (x[..., 5:] for x in qkv.split((14, 3, 3), dim=1))
    nb = fo.block_bytes(8, 128)
    both = torch.full((5, 2, 3, nb), 9, dtype=torch.uint8, device="cuda")  # a block's K and V side by side
    pools, before = (both[:, 0], both[:, 1]), (both[:, 0].cpu(), both[:, 1].cpu())
    ids, offsets = _slots(7, 5, 8, 5)
    positions, table = torch.arange(7, device="cuda", dtype=torch.int32), _table(7, 128)
    buffer = torch.zeros(7, 30, 140, device="cuda", dtype=HALF)
    q_out = buffer[:, 1:29:2, 3:131]
    got = fd.fused_rope_kv_append_fp4(q, k, v, *pools, ids, offsets, positions, cos_sin_table=table, q_out=q_out)
    assert got is q_out
    _check(q, k, v, pools, before, ids, offsets, 8, q_out, table, positions, 128)
    untouched = torch.ones_like(buffer, dtype=torch.bool)
    untouched[:, 1:29:2, 3:131] = False
    assert not bool(buffer[untouched].any())
    heads = torch.full((3, 5, nb), 9, dtype=torch.uint8, device="cuda").transpose(0, 1)  # heads ahead of blocks
    other = torch.full((3, 5, nb), 9, dtype=torch.uint8, device="cuda").transpose(0, 1)
    fd.fused_rope_kv_append_fp4(q, k, v, heads, other, ids, offsets, positions, cos_sin_table=table)
    assert torch.equal(heads, pools[0]) and torch.equal(other, pools[1])
    k_out = torch.zeros(7, 6, 128, device="cuda", dtype=BF)[:, ::2]
    v_out = torch.zeros(3 * 7 * 128 + 1, device="cuda", dtype=BF)[1:].view(3, 7, 128).transpose(0, 1)
    fd.paged_kv_read_fp4_into(*pools, ids, offsets, k_out, v_out)
    at = ids.cpu(), slice(None), offsets.cpu()
    assert torch.equal(k_out.cpu().double(), fo.unpack(pools[0], 8, 128, False)[at])
    assert torch.equal(v_out.cpu().double(), fo.unpack(pools[1], 8, 128, True)[at])


def test_refusals_that_need_a_gpu():
    q, k, v = (x.contiguous() for x in _tokens(4, 4, 2, 64, BF, 1))
    pools = _pools(2, 2, 8, 64)
    ids, offsets = _slots(4, 2, 8, 1)
    with pytest.raises(ValueError, match="must lie apart"):
        fd.fused_rope_kv_append_fp4(q, k, v, *pools, ids, offsets, ids, q_out=q)
    with pytest.raises(ValueError, match="different tensors"):
        fd.kv_append_fp4(k, v, pools[0], pools[0], ids, offsets)
    with pytest.raises(ValueError, match="different tensors"):
        fd.paged_kv_read_fp4_into(*pools, ids, offsets, k, k)
    with pytest.raises(ValueError, match="same CUDA device"):
        fd.kv_append_fp4(k, v, *pools, ids.cpu(), offsets)
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        fd.kv_append_fp4(k, v, pools[0], pools[1].cpu(), ids, offsets)
    flat = torch.zeros(2 * 2 * 272 + 8, dtype=torch.uint8, device="cuda")
    off = flat[8:].view(2, 2, 272)
    fd.kv_append_fp4(k, v, *pools, ids, offsets)
    with pytest.raises(ValueError, match="16-byte lines"):
        fd.kv_append_fp4(k, v, pools[0], off, ids, offsets)  # the kept call's shapes and strides
    empty = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert fd.fused_rope_kv_append_fp4(q[:0], k[:0], v[:0], *pools, empty, empty, empty).shape == (0, 4, 64)
    fd.kv_append_fp4(k[:0], v[:0], *pools, empty, empty)
    assert fd.paged_kv_read_fp4(*pools, empty, empty, 64)[0].shape == (0, 2, 64)


def test_append_and_read_in_a_graph_and_on_another_stream():
    q, k, v = _tokens(40, 16, 2, 128, BF, 6)
    table, positions = _table(300, 128), torch.arange(40, device="cuda")
    ids, offsets = _slots(40, 9, 16, 6)
    pools, want = _pools(9, 2, 16, 128), _pools(9, 2, 16, 128)
    q_out, k_out, v_out = torch.zeros(40, 16, 128, device="cuda", dtype=BF), *(torch.zeros(40, 2, 128, device="cuda", dtype=BF)
                                                                               for _ in range(2))

    def step():
        fd.fused_rope_kv_append_fp4(q, k, v, *pools, ids, offsets, positions, cos_sin_table=table, q_out=q_out,
                                    check_indices=False)
        fd.paged_kv_read_fp4_into(*pools, ids, offsets, k_out, v_out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        q.normal_()
        k.normal_()
        positions += 30 * i
        graph.replay()
        torch.cuda.synchronize()
        expect = fd.fused_rope_kv_append_fp4(q, k, v, *want, ids, offsets, positions, cos_sin_table=table)
        assert torch.equal(q_out, expect) and torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1])
        assert torch.equal(k_out.cpu().double(), fo.unpack(pools[0], 16, 128, False)[ids.cpu(), :, offsets.cpu()])
        assert torch.equal(v_out.cpu().double(), fo.unpack(pools[1], 16, 128, True)[ids.cpu(), :, offsets.cpu()])


def test_slots_past_four_gigabytes():
    nb = fo.block_bytes(32, 128)
    blocks = (1 << 32) // (8 * nb) + 40
    pools = [torch.empty((blocks, 8, nb), dtype=torch.uint8, device="cuda") for _ in range(2)]
    q, k, v = _tokens(20, 8, 8, 128, BF, 2)
    ids = torch.arange(blocks - 20, blocks, device="cuda")
    offsets = torch.arange(20, device="cuda")
    fd.kv_append_fp4(k, v, *pools, ids, offsets)
    small = _pools(20, 8, 32, 128)
    fd.kv_append_fp4(k, v, *small, ids - (blocks - 20), offsets)
    near = fd.paged_kv_read_fp4(*small, ids - (blocks - 20), offsets, 128)
    for got, want in zip(fd.paged_kv_read_fp4(*pools, ids, offsets, 128), near):
        assert torch.equal(got, want)
    assert np.isfinite(near[0].float().cpu().numpy()).all()


def test_q_out_next_to_q_in_one_buffer():
    """Each token's rotated heads behind its others, or every second head: no element is shared."""
    q, k, v = (x.contiguous() for x in _tokens(9, 8, 2, 128, BF, 11))
    ids, offsets = _slots(9, 3, 8, 11)
    positions = torch.arange(9, device="cuda")
    want = fd.fused_rope_kv_append_fp4(q, k, v, *_pools(3, 2, 8, 128), ids, offsets, positions)
    for first, second in ((slice(0, 8), slice(8, 16)), (slice(0, 16, 2), slice(1, 16, 2))):
        buffer = torch.zeros(9, 16, 128, device="cuda", dtype=BF)
        buffer[:, first] = q
        for _ in range(2):
            fd.fused_rope_kv_append_fp4(buffer[:, first], k, v, *_pools(3, 2, 8, 128), ids, offsets, positions,
                                        q_out=buffer[:, second])
            assert torch.equal(buffer[:, second], want) and torch.equal(buffer[:, first], q)
        with pytest.raises(ValueError, match="must lie apart"):
            fd.fused_rope_kv_append_fp4(buffer[:, :8], k, v, *_pools(3, 2, 8, 128), ids, offsets, positions, q_out=buffer[:, 4:12])


def test_q_out_over_k_or_v_is_refused():
    """Other workgroups still read them."""
    q, k, v = (x.contiguous() for x in _tokens(5, 4, 4, 128, BF, 12))
    pools = _pools(2, 4, 8, 128)
    before = [p.clone() for p in pools]
    ids, offsets = _slots(5, 2, 8, 12)
    qkv = torch.cat((q, k, v), dim=1)
    parts = qkv.split(4, dim=1)
    for args, q_out in (((q, k, v), k), ((q, k, v), v), (parts, qkv[:, 6:10]), (parts, qkv[:, 8:])):
        for _ in range(2):
            with pytest.raises(ValueError, match="must lie apart from q, k and v"):
                fd.fused_rope_kv_append_fp4(*args, *pools, ids, offsets, ids, q_out=q_out)
    assert all(torch.equal(p, b) for p, b in zip(pools, before)) and torch.equal(qkv, torch.cat((q, k, v), dim=1))
    wide = torch.cat((qkv, torch.zeros_like(q)), dim=1)
    parts = wide[:, :12].split(4, dim=1)
    got = fd.fused_rope_kv_append_fp4(*parts, *pools, ids, offsets, ids, q_out=wide[:, 12:])
    assert torch.equal(got, fd.fused_rope_kv_append_fp4(q, k, v, *before, ids, offsets, ids))


def test_caches_that_share_blocks_are_refused():
    _, k, v = _tokens(4, 1, 2, 64, BF, 13)
    ids, offsets = _slots(4, 4, 8, 13)
    pool = torch.zeros((10, 2, fo.block_bytes(8, 64)), dtype=torch.uint8, device="cuda")
    for k_cache, v_cache in ((pool[:6], pool[4:]), (pool[4:], pool[:6]), (pool[::2], pool[4:9]), (pool[:6], pool[:6])):
        for _ in range(2):
            with pytest.raises(ValueError, match="share no element"):
                fd.kv_append_fp4(k, v, k_cache, v_cache, ids, offsets)
            with pytest.raises(ValueError, match="share no element"):
                fd.fused_rope_kv_append_fp4(k, k, v, k_cache, v_cache, ids, offsets, ids)
    assert not bool(pool.any())
    want = _pools(5, 2, 8, 64, 0)
    fd.kv_append_fp4(k, v, *want, ids, offsets)
    for pair in ((pool[:5], pool[5:]), (pool[5:], pool[:5]), (pool[::2], pool[1::2]), (pool[1::2], pool[::2])):
        pool.zero_()
        fd.kv_append_fp4(k, v, *pair, ids, offsets)
        assert all(torch.equal(a, b) for a, b in zip(pair, want))


def test_outputs_of_the_read_that_share_tokens_are_refused():
    pools = [fo.random_pool(3, 2, 8, 64, 14 + i, bool(i)).cuda() for i in range(2)]
    ids, offsets = _slots(6, 3, 8, 14)
    buffer = torch.zeros(6, 6, 64, device="cuda", dtype=BF)
    for k_out, v_out in ((buffer[:, :2], buffer[:, 1:3]), (buffer[:, 2:4], buffer[:, 1:3]), (buffer[:, :3:2], buffer[:, 2:4])):
        for _ in range(2):
            with pytest.raises(ValueError, match="share no element"):
                fd.paged_kv_read_fp4_into(*pools, ids, offsets, k_out, v_out)
    assert not bool(buffer.any())
    want = fd.paged_kv_read_fp4(*pools, ids, offsets, 64)
    for outs in ((buffer[:, :2], buffer[:, 2:4]), (buffer[:, 4:], buffer[:, 1:3]), (buffer[:, :4:2], buffer[:, 1:4:2])):
        buffer.zero_()
        got = fd.paged_kv_read_fp4_into(*pools, ids, offsets, *outs)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and int(buffer.any(dim=2).any(dim=0).sum()) == 4


@pytest.mark.parametrize("heads, d, n", [(2, 64, 7), (3, 128, 300), (8, 128, 4099)])
@pytest.mark.parametrize("shift", [1, 2, 3, 5])
def test_reads_into_rows_off_the_16_byte_lines(heads, d, n, shift):
    """Outputs that begin anywhere, with rows of odd pitch; what lies between them stays as it was."""
    pools = [fo.random_pool(20, heads, 16, d, 5 + i, bool(i)).cuda() for i in range(2)]
    gen = torch.Generator().manual_seed(n)
    ids, offsets = torch.randint(0, 20, (n,), generator=gen).cuda(), torch.randint(0, 16, (n,), generator=gen).cuda()
    want = fd.paged_kv_read_fp4(*pools, ids, offsets, d)
    wide = [torch.full((n, heads, d + 5 + 2 * i), 3.0, device="cuda", dtype=BF) for i in range(2)]
    outs = [w[..., shift : shift + d] for w in wide]
    for got, expect, w in zip(fd.paged_kv_read_fp4_into(*pools, ids, offsets, *outs), want, wide):
        assert torch.equal(got, expect)
        assert bool((w[..., :shift] == 3).all()) and bool((w[..., shift + d :] == 3).all())
