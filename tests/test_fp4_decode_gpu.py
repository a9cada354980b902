"""GPU parity of decode over a 4-bit cache against its plain 64-bit form (tests/fp4_oracle.py).

Tolerances, by arithmetic.  Let u be half a step of q's type, relative to a value (bf16 2^-8, fp16 2^-11), e = 2^-24 that
of fp32, x a token's score times log2 e, and d a bound on the error of x.

* The cache's values are exact, and so is every product of a query's and a key's value (11 and 2 bits).  A dot product of
  D terms summed in fp32 in any order is off by at most (D - 1) e sum |q k|; the scale's rounding and product add 3 e |x|.
  A query held as a sum of 8-bit terms keeps each value to 2^-21 of the largest of its 32 dims.  So
  d <= scale log2(e) ((D + 2) e max sum |q k| + 2^-21 max sum (largest |q| of 32) |k|).
* A probability 2^(x - M) / L is off, relatively, by 2 d ln 2 and by what the arithmetic adds: the exponentials' arguments
  (below 2^8 where they count) are rounded by 2^-16 at each of at most three levels, v_exp_f32 and v_rcp_f32 by 2^-22,
  and the sums of n <= 2^15 positive terms by 2^-16: 2^-13 in all.
* out = sum p v: the probabilities enter the product rounded to q's type or better (u), the result leaves rounded (u):
  with A = sum p |v|, |error| <= (u + 2 d + 2^-13) A + u |out|, plus one smallest step.
"""

import math
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

import flashdec_amd as fd
from flashdec_amd import _lib
from tests import fp4_oracle as fo

pytestmark = pytest.mark.gpu

BF, HALF = torch.bfloat16, torch.float16
E = 2.0**-24
HALF_STEP = {BF: 2.0**-8, HALF: 2.0**-11}
SMALLEST = {BF: 2.0**-126, HALF: 2.0**-24}
EDGES = [700, 3, 0, 129, 2000, 64, 31, 1, 33, 32, 95, 511]


def _inputs(lens, hq, hkv, d, block, dtype, seed=1, index=torch.int32, width=None, spread=3):
    need = [-(-max(n, 0) // block) for n in lens]
    blocks = sum(need) + 3
    gen = torch.Generator().manual_seed(seed)
    order = torch.randperm(blocks, generator=gen)
    table = torch.full((len(lens), width or max(1, *need)), -1, dtype=index)
    for b, row in enumerate(order[: sum(need)].split(need)):
        table[b, : len(row)] = row
    q = (2 * torch.randn(len(lens), hq, d, generator=gen)).to(dtype)
    k, v = (fo.random_pool(blocks, hkv, block, d, seed + i, bool(i), spread) for i in range(2))
    return q.cuda(), k.cuda(), v.cuda(), table.cuda(), torch.tensor(lens, dtype=index).cuda()


def _check(out, q, k, v, table, lens, block, scale=None):
    d = q.shape[2]
    keys, values = fo.unpack(k, block, d, False), fo.unpack(v, block, d, True)
    want, size, most, split = fo.attend(q, keys, values, table, lens, scale)
    factor = math.log2(math.e) * (1.0 / math.sqrt(d) if scale is None else abs(scale))
    off = factor * ((d + 2) * E * most + 2.0**-21 * split)
    u = HALF_STEP[q.dtype]
    got = out.detach().cpu().double()
    bound = (u + 2 * off + 2.0**-13) * size + u * want.abs() + SMALLEST[q.dtype]
    assert torch.equal(got.isnan(), want.isnan())
    worst = ((got - want).abs() - bound).nan_to_num(-1.0).max()
    assert float(worst) <= 0, f"off by {float((got - want).abs().nan_to_num(0).max()):.3g}, over by {float(worst):.3g}"


@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("hq, hkv, d, block", [(16, 2, 128, 16), (16, 2, 128, 32), (8, 8, 128, 8), (14, 2, 64, 16),
                                               (32, 8, 64, 32), (6, 1, 64, 8), (12, 4, 128, 32)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_decode(dtype, hq, hkv, d, block, index):
    q, k, v, table, lens = _inputs(EDGES, hq, hkv, d, block, dtype, index=index)
    _check(fd.paged_decode_attention_fp4(q, k, v, table, lens), q, k, v, table, lens, block)


@pytest.mark.parametrize("hq, hkv", [(17, 1), (32, 1), (40, 2), (71, 1), (300, 1)])
def test_groups_past_sixteen_heads(hq, hkv):
    for d, dtype in ((128, BF), (64, HALF)):
        q, k, v, table, lens = _inputs([300, 1, 0, 77], hq, hkv, d, 16, dtype)
        _check(fd.paged_decode_attention_fp4(q, k, v, table, lens), q, k, v, table, lens, 16)


@pytest.mark.parametrize("lens", [[1], [16], [17], [100], [4097], [20000], [1] * 300, [40] * 70, [9000, 0, 3, 12000] * 3])
@pytest.mark.parametrize("d, dtype", [(128, BF), (64, HALF)])
def test_batches_of_other_plans(lens, d, dtype):
    q, k, v, table, lens = _inputs(lens, 8, 2, d, 32, dtype)
    _check(fd.paged_decode_attention_fp4(q, k, v, table, lens), q, k, v, table, lens, 32)


@pytest.mark.parametrize("lens, hq, hkv, tiles", [
    ([4000, 37, 0, 900, 1, 2050, 33, 128], 16, 2, 256), ([0] * 63 + [8100], 4, 2, 256), ([5] + [0] * 5, 16, 8, 128),
    ([1, 0, 31, 32, 33, 64, 65] * 9 + [3000], 8, 2, 100), ([700], 8, 1, 4096), ([0, 0], 8, 2, 1100),
    ([20000, 1], 4, 4, 700), ([3000, 100, 0, 513], 40, 1, 512), ([2048] * 16, 8, 4, 64)])
@pytest.mark.parametrize("d, dtype, block", [(128, BF, 32), (64, HALF, 16), (128, HALF, 8)])
def test_long_tables_of_rows_of_any_length(lens, hq, hkv, tiles, d, dtype, block):
    """Few rows and heads and wide tables: chunks are cut by the rows' own lengths."""
    q, k, v, table, lens = _inputs(lens, hq, hkv, d, block, dtype, width=32 * tiles // block, index=torch.int64)
    both = torch.stack((lens, lens + 1), dim=1)
    out = torch.full_like(q, math.nan)
    _check(fd.paged_decode_attention_fp4_into(q, k, v, table, both[:, 0], out), q, k, v, table, lens, block)
    _check(fd.paged_decode_attention_fp4(q, k, v, table, lens, ragged=True), q, k, v, table, lens, block)


@pytest.mark.parametrize("lens, hq, hkv, tiles", [
    ([1500, 0, 31, 2048, 5, 700, 64, 33] * 6 + [2048, 0], 16, 8, 64), ([1024] * 40, 8, 8, 64), ([0] * 63 + [1], 8, 8, 64),
    ([400] * 65, 4, 4, 64), ([700, 0, 33, 5, 64, 0, 0] * 20, 4, 2, 64), ([0] * 255 + [900], 4, 2, 32),
    ([3, 40] * 128 + [1000], 4, 2, 32), ([900, 30], 4, 4, 32), ([40, 7, 0] * 15, 20, 1, 2), ([64, 0, 90, 1] * 10, 64, 64, 32)])
@pytest.mark.parametrize("d, dtype, block", [(128, BF, 32), (64, HALF, 16)])
def test_ragged_batches(lens, hq, hkv, tiles, d, dtype, block):
    """Batches whose rows have a workgroup each or more, and such that are too short or too many to be cut."""
    q, k, v, table, lens = _inputs(lens, hq, hkv, d, block, dtype, width=32 * tiles // block)
    out = torch.full_like(q, math.nan)
    _check(fd.paged_decode_attention_fp4_into(q, k, v, table, lens, out, ragged=True), q, k, v, table, lens, block)


def test_captured_rows_that_grow_in_long_tables():
    """A replay cuts its chunks by the lengths that it finds; lengths outside the table are its ends."""
    q, k, v, table, lens = _inputs([8000, 100, 1, 3000], 16, 4, 128, 32, BF, width=320)
    table[:] = torch.randint(0, k.shape[0], table.shape, device="cuda")
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    fd.paged_decode_attention_fp4_into(q, k, v, table, lens, out)
    with torch.cuda.graph(graph):
        fd.paged_decode_attention_fp4_into(q, k, v, table, lens, out)
    for new in ([8000, 100, 1, 3000], [1, 10000, 0, 17], [0, 0, 0, 0], [10240, 10240, 10240, 10240], [-3, 2**31 - 1, 0, 64]):
        lens.copy_(torch.tensor(new))
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        _check(out, q, k, v, table, lens, 32)
        assert torch.equal(out, fd.paged_decode_attention_fp4(q, k, v, table, lens))


@pytest.mark.parametrize("lens", [[100], [100, 0, 70000], [33] * 64])
def test_the_widest_tables(lens):
    """Tables of nearly 2^31 tokens: no place in one is past 32 bits, wherever a chunk would begin."""
    q, k, v, _, _ = _inputs([32], 8, 1, 128, 32, BF)
    q = torch.randn(len(lens), 8, 128, device="cuda").to(BF)
    table = torch.ones(1, 1, dtype=torch.int32, device="cuda").expand(len(lens), (2**31 - 5000) // 32)
    lens = torch.tensor(lens, device="cuda")
    short = table[:, : (int(lens.max()) + 31) // 32].contiguous()
    for ragged in (False, True):
        _check(fd.paged_decode_attention_fp4(q, k, v, table, lens, ragged=ragged), q, k, v, short, lens, 32)


def test_rows_of_a_wide_table_and_lengths_past_it():
    q, k, v, table, lens = _inputs([100, 64, 1, 64], 16, 2, 128, 16, BF, width=400)
    lens[0], lens[1] = -5, 2**31 - 1
    _check(fd.paged_decode_attention_fp4(q, k, v, table, lens), q, k, v, table, lens, 16)
    q, k, v, table, lens = _inputs([100, 64], 16, 2, 128, 16, BF)
    lens[:] = 1000
    _check(fd.paged_decode_attention_fp4(q, k, v, table, lens), q, k, v, table, lens, 16)


@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize("d, dtype", [(128, BF), (64, HALF)])
def test_blocks_outside_the_pool_are_not_attended(block, d, dtype):
    q, k, v, table, lens = _inputs([400, 130, 70], 8, 2, d, block, dtype)
    table[0, 1], table[0, 4], table[1, 0] = -1, k.shape[0], -7
    table[2] = 2**30
    out = fd.paged_decode_attention_fp4(q, k, v, table, lens)
    _check(out, q, k, v, table, lens, block)
    assert not bool(out[2].any())


@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize("d, dtype", [(128, BF), (64, HALF)])
def test_what_lies_behind_a_rows_end_does_not_count(block, d, dtype):
    """Every byte that holds no attended token is 255: NaN scales and the largest codes."""
    q, k, v, table, lens = _inputs(EDGES, 8, 2, d, block, dtype)
    want = fd.paged_decode_attention_fp4(q, k, v, table, lens)
    seen = torch.zeros(k.shape[0], block, dtype=torch.bool)
    for b, n in enumerate(lens.tolist()):
        at = torch.arange(n)
        seen[table[b].cpu().long()[at // block], at % block] = True
    for pool, values in ((k, False), (v, True)):
        code_at, _, scale_at = fo.places(block, d, values)
        live = torch.zeros(pool.shape[0], pool.shape[2], dtype=torch.bool)
        for tok in range(block):
            for at in (code_at[tok], scale_at[tok]):
                live[:, at] |= seen[:, tok, None]
        pool.copy_(torch.where(live.cuda()[:, None], pool, 255))
    got = fd.paged_decode_attention_fp4(q, k, v, table, lens)
    assert torch.equal(got, want)


@pytest.mark.parametrize("d, dtype", [(128, BF), (64, HALF)])
def test_nan_groups(d, dtype):
    """A NaN key gives its rows NaN, a NaN value group the dims of its group; others stay as they are."""
    q, k, v, table, lens = _inputs([200, 77, 300], 8, 2, d, 16, dtype)
    block = 16
    at = fo.places(block, d, False)[2], fo.places(block, d, True)[2]
    k[table[0, 3].long(), 1, at[0][5, 1]] = 255
    v[table[2, 2].long(), 0, at[1][7, 0]] = 255
    out = fd.paged_decode_attention_fp4(q, k, v, table, lens)
    _check(out, q, k, v, table, lens, block)
    nan = out.isnan().cpu()
    assert bool(nan[0, 4:].all()) and bool(nan[2, :4, :32].all()) and int(nan.sum()) == 4 * d + 4 * 32


@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("d", [64, 128])
def test_odd_queries(dtype, d):
    """Zeros, values far apart within a group, the type's ends, infinities and NaN."""
    q, k, v, table, lens = _inputs([150] * 6, 8, 2, d, 16, dtype)
    q[0] = 0.0
    q[1, :, ::32] *= 2.0**12  # (the others lie far below their group's largest)
    q[2] *= 2.0**-13
    q[3, :, 1::2] = 0.0
    q[4, 0, 5], q[4, 5, 40] = math.nan, math.inf
    q[5] = torch.finfo(dtype).tiny / 4
    out = fd.paged_decode_attention_fp4(q, k, v, table, lens)
    nan = out[4].isnan().cpu()
    assert bool(nan[0].all()) and bool(nan[5].all()) and int(nan.sum()) == 2 * d
    keep = [0, 1, 2, 3, 5]
    _check(out[keep], q[keep], k, v, table[keep], lens[keep], 16)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 0.02])
def test_scales(scale):
    q, k, v, table, lens = _inputs(EDGES, 16, 2, 128, 32, BF, spread=1)
    q *= 0.25
    out = fd.paged_decode_attention_fp4(q, k, v, table, lens, sm_scale=scale)
    _check(out, q, k, v, table, lens, 32, scale)


@pytest.mark.parametrize("base", [5, 60, 120])
def test_scale_bytes_far_from_one(base):
    """Values from 2^-120 to 2^118: the products' range is that of 32-bit numbers."""
    q, k, v, table, lens = _inputs([300, 20], 8, 2, 128, 16, BF)
    part = v[:, :, 16 * 64 :]
    part.copy_((part.int() - 125 + base + 0).clamp(2, 252).to(torch.uint8))
    _check(fd.paged_decode_attention_fp4(q, k, v, table, lens), q, k, v, table, lens, 16)
    part.copy_((part.int() - base + 245).clamp(2, 250).to(torch.uint8))
    _check(fd.paged_decode_attention_fp4(q, k, v, table, lens), q, k, v, table, lens, 16)


@pytest.mark.parametrize("d, dtype", [(128, BF), (64, HALF)])
def test_views(d, dtype):
    """q and out of any strides and alignment, pools of other orders, index tensors with strides."""
    q, k, v, table, lens = _inputs(EDGES, 8, 2, d, 16, dtype)
    want = fd.paged_decode_attention_fp4(q, k, v, table, lens)
    wide = torch.zeros(len(EDGES), 8, 2 * d + 3, device="cuda", dtype=dtype)
    strided, odd = wide[:, :, 1 : 2 * d + 1 : 2], wide[:, :, 3 : d + 3]
    out = torch.zeros(8, d, len(EDGES), device="cuda", dtype=dtype).permute(2, 0, 1)
    for view in (strided, odd):
        view.copy_(q)
        assert torch.equal(fd.paged_decode_attention_fp4_into(view, k, v, table, lens, out), want)
    both = torch.stack((k, v), dim=1)
    heads = (torch.stack((k, v), dim=0).transpose(1, 2).contiguous().transpose(1, 2))
    tables = torch.stack((table, table - 1), dim=2)[..., 0]
    lengths = torch.stack((lens, lens + 1), dim=1)[:, 0]
    for k2, v2 in ((both[:, 0], both[:, 1]), heads):
        assert torch.equal(fd.paged_decode_attention_fp4(q, k2, v2, tables, lengths), want)
    buffer = torch.zeros(len(EDGES) * 8 * d + 1, device="cuda", dtype=dtype)
    off = buffer[1:].view(len(EDGES), 8, d)
    assert torch.equal(fd.paged_decode_attention_fp4_into(q, k, v, table, lens, off), want)
    assert torch.equal(fd.paged_decode_attention_fp4(q, k, v, table, lens, kv_reuse=True), want)
    assert torch.equal(fd.paged_decode_attention_fp4(q, k, v, table, lens, sm_scale=torch.tensor(1 / math.sqrt(d))), want)


def test_rows_that_share_blocks():
    q, k, v, table, lens = _inputs([320] * 5, 16, 2, 128, 32, BF)
    table[1:, :8] = table[0, :8]
    for reuse in (False, True):
        _check(fd.paged_decode_attention_fp4(q, k, v, table, lens, kv_reuse=reuse), q, k, v, table, lens, 32)


def test_captured_calls_and_streams():
    """Two captured calls of different sizes and eager ones in between, each with its own partials."""
    first = _inputs([5000, 300], 8, 2, 128, 32, BF, seed=3)
    second = _inputs([900] * 9, 16, 2, 64, 16, HALF, seed=4)
    outs = [torch.zeros_like(first[0]), torch.zeros_like(second[0])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for call, out in zip((first, second), outs):
            fd.paged_decode_attention_fp4_into(*call, out)
    torch.cuda.synchronize()
    graphs = []
    for call, out in zip((first, second), outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            fd.paged_decode_attention_fp4_into(*call, out)
    for i in range(4):
        for call, out, graph in zip((first, second), outs, graphs):
            call[0].normal_()
            out.zero_()
            if i % 2:
                call[4].sub_(1)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for call, out in zip((first, second), outs):
            assert torch.equal(out, fd.paged_decode_attention_fp4(*call))


def test_threads_on_one_stream():
    """Calls of several threads at once: each has its own partials."""
    jobs = [_inputs(lens, 8, 2, d, 16, dtype, seed=i) for i, (lens, d, dtype) in enumerate(
        (([3000] * 3, 128, BF), ([7, 900], 64, HALF), ([20000], 128, BF)))]
    want = [fd.paged_decode_attention_fp4(*j) for j in jobs]
    torch.cuda.synchronize()
    with ThreadPoolExecutor(3) as pool:
        got = [[f.result(timeout=60) for f in [pool.submit(fd.paged_decode_attention_fp4, *j) for j in jobs]]
               for _ in range(20)]
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_calls_of_different_sizes_in_turn():
    calls = [_inputs(lens, 8, 2, d, 16, dtype, seed=i) for i, (lens, d, dtype) in enumerate(
        (([40], 128, BF), ([3000] * 3, 128, BF), ([7, 900], 64, HALF), ([1] * 40, 128, BF)))]
    want = []
    for q, k, v, table, lens in calls:  # (a workspace that grows between kept calls of other operators)
        fd.paged_kv_read_fp4(k, v, table[0, :1].long(), torch.zeros_like(table[0, :1]), q.shape[2])
        want.append(fd.paged_decode_attention_fp4(q, k, v, table, lens))
    for _ in range(3):
        for call, w in zip(calls, want):
            assert torch.equal(fd.paged_decode_attention_fp4(*call), w)


def test_refusals():
    q, k, v, table, lens = _inputs([40, 8], 4, 2, 64, 16, BF)
    dec = fd.paged_decode_attention_fp4
    for args, message in (
            ((q.float(), k, v, table, lens), "float16 and bfloat16"), ((q[0], k, v, table, lens), "shape"),
            ((q[:, :3], k, v, table, lens), "divisible"), ((q, k[:, :1], v, table, lens), "same shape"),
            ((q, k.float(), v, table, lens), "uint8"), ((q, k, v, table.float(), lens), "int32 or int64"),
            ((q, k, v, table, lens.short()), "int32 or int64"), ((q, k, v, table[:1], lens), "one row/value"),
            ((q, k, v, table, lens[:1]), "one row/value"), ((q, k, v, table[:, :0], lens), "max_blocks_per_seq"),
            ((q[:0], k, v, table[:0], lens[:0]), "positive"), ((q, k.cpu(), v, table, lens), "CUDA"),
            ((q, k, v, table.cpu(), lens), "CUDA"), ((q.new_zeros(2, 4, 96), k, v, table, lens), "head_dim")):
        with pytest.raises(ValueError, match=message):
            dec(*args)
    for bad in (q.new_zeros(2, 4, 32), q.half(), q[:1].expand(2, 4, 64)):
        with pytest.raises(ValueError, match="out must"):
            fd.paged_decode_attention_fp4_into(q, k, v, table, lens, bad)
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        dec(q, k, v, table, [40, 8])
    dec(q, k, v, table, lens)
    flat = torch.zeros(k.numel() + 8, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="16-byte lines"):
        dec(q, flat[8:].view_as(k), v, table, lens)


def test_caches_past_four_gigabytes():
    q, k, v, table, lens = _inputs([500, 100], 8, 2, 128, 32, BF)
    blocks = (1 << 32) // (2 * k.shape[2]) + k.shape[0]
    pools = []
    for small in (k, v):
        pool = torch.empty((blocks, 2, k.shape[2]), dtype=torch.uint8, device="cuda")
        pool[blocks - k.shape[0] :] = small
        pools.append(pool)
    far = torch.where(table < 0, table, table + (blocks - k.shape[0]))
    assert torch.equal(fd.paged_decode_attention_fp4(q, *pools, far, lens), fd.paged_decode_attention_fp4(q, k, v, table, lens))


def test_append_then_decode():
    """A prompt and some steps through the cache: attention over what was appended, quantised."""
    hq, hkv, d, block, start, steps = 16, 2, 128, 16, 45, 6
    gen = torch.Generator().manual_seed(7)
    pools = [torch.full((12, hkv, fo.block_bytes(block, d)), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
    table = torch.randperm(12, generator=gen)[:8].view(2, 4).cuda()
    mirror = [p.cpu() for p in pools]
    lens = torch.tensor([start, start - 20], device="cuda")
    for step in range(-1, steps):
        new = [torch.arange(int(n)) for n in lens] if step < 0 else [torch.tensor([int(n)]) for n in lens]
        row = torch.cat([torch.full_like(x, b) for b, x in enumerate(new)]).cuda()
        at = torch.cat(new).cuda()
        q, k, v = (torch.randn(len(at), h, d, generator=gen).to(BF).cuda() for h in (hq, hkv, hkv))
        ids, offsets = table[row, at // block], at % block
        rotated = fd.fused_rope_kv_append_fp4(q, k, v, *pools, ids, offsets, at)
        whole = [torch.zeros(12, hkv, block, d, dtype=torch.float32, device="cuda") for _ in range(2)]
        fd.fused_rope_kv_append(q.float(), k.float(), v.float(), *whole, ids, offsets, at)
        for m, cache, values in zip(mirror, whole, (False, True)):
            fo.store(m, ids.cpu(), offsets.cpu(), cache[ids, :, offsets], block, values)
        if step >= 0:
            lens += 1
            out = fd.paged_decode_attention_fp4(rotated, *pools, table, lens)
            assert torch.equal(pools[0].cpu(), mirror[0]) and torch.equal(pools[1].cpu(), mirror[1])
            _check(out, rotated, *(m.cuda() for m in mirror), table, lens, block)


def test_launches_are_recorded():
    q, k, v, table, lens = _inputs([40, 8], 4, 2, 64, 16, BF)
    _lib.record_launches()
    try:
        fd.paged_decode_attention_fp4(q, k, v, table, lens)
        assert any("fp4_decode" in name for name in _lib.last_launch())
    finally:
        _lib.record_launches(False)


@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize("d, dtype", [(128, BF), (64, HALF)])
@pytest.mark.parametrize("tokens", [None, 8192])
def test_ids_past_32_bits_are_outside_the_pool(block, d, dtype, tokens):
    """Also where the table is wide and chunks are cut by the rows' lengths."""
    q, k, v, table, lens = _inputs([400, 130, 70], 8, 2, d, block, dtype, index=torch.int64, width=tokens and tokens // block)
    table[0, 1] += 2**32  # (the low words stay as they are)
    table[0, 4] -= 2**32
    table[1, 0] += 5 * 2**32
    _check(fd.paged_decode_attention_fp4(q, k, v, table, lens), q, k, v, table, lens, block)


@pytest.mark.parametrize("dtype", [BF, HALF])
@pytest.mark.parametrize("tokens", [64, 5000])
@pytest.mark.parametrize("d", [64, 128])
def test_probabilities_keep_more_bits_than_the_operands(dtype, d, tokens):
    """Two kinds of tokens in turn, whose probabilities are apart by less than half a step of bf16, with the values 1 and -1:
    rounded to bf16 the probabilities are equal and the result is zero, where it is as much as a quarter of that step.  In two
    terms each is off by at most 2^-16 of itself (half a step of half a step), in place of the first bound's u."""
    block = 32
    q, k, v, table, lens = _inputs([tokens] * 4, 2, 1, d, block, dtype)
    k.zero_()
    v.zero_()
    key_code, _, key_scale = fo.places(block, d, False)
    value_code, _, value_scale = fo.places(block, d, True)
    k[..., key_scale.flatten()] = 127
    v[..., value_scale.flatten()] = 127
    v[:, :, value_code[::2].flatten()] = 0x22  # two dims of 1
    v[:, :, value_code[1::2].flatten()] = 0xAA  # of -1
    k[:, :, key_code[1::2, 0]] = 0x02  # 1 in the first dim
    q.zero_()
    q[:, :, 0] = torch.tensor([0.45, 0.35, -0.4, -0.3])[:, None] * 2.0**-8
    out = fd.paged_decode_attention_fp4(q, k, v, table, lens, sm_scale=1.0)
    keys, values = fo.unpack(k, block, d, False), fo.unpack(v, block, d, True)
    want, size, most, split = fo.attend(q, keys, values, table, lens, 1.0)
    assert float(want.abs().min()) > 2.0**-11
    off = math.log2(math.e) * ((d + 2) * E * most + 2.0**-21 * split)
    bound = (2.0**-16 + 2 * off + 2.0**-13) * size + HALF_STEP[dtype] * want.abs() + SMALLEST[dtype]
    assert float(((out.cpu().double() - want).abs() - bound).max()) <= 0


@pytest.mark.parametrize("dtype, d", [(BF, 128), (BF, 64), (HALF, 128), (HALF, 64)])
@pytest.mark.parametrize("tokens", [70, 6000])
@pytest.mark.parametrize("size", [4, 13, 20, 27, 60])
def test_scores_far_beyond_a_32_bit_numbers_steps(dtype, d, tokens, size):
    """Queries of 1000 to 60000 and keys up to 6 * 2^size: the largest score is thousands above the next, as products of
    exactly known numbers, and its token has all of the weight, whatever a step of the scores is."""
    block, hq = 16, 8
    q, k, v, table, lens = _inputs([tokens] * 3, hq, 1, d, block, dtype, spread=1)
    k.zero_()
    code_at, _, scale_at = fo.places(block, d, False)
    k[..., scale_at.flatten()] = 127 + size
    k[..., code_at[:, 0]] = 0x06  # 4 in the first dim of every token
    best = torch.tensor([0, tokens // 2, tokens - 1])
    for b, t in enumerate(best.tolist()):
        k[table[b, t // block].long(), 0, code_at[t % block, 0]] = 0x07  # 6
    q.zero_()
    gen = torch.Generator().manual_seed(size)
    q[:, :, 0] = (1000 + 59000 * torch.rand(3, hq, generator=gen)).to(dtype).cuda()
    out = fd.paged_decode_attention_fp4(q, k, v, table, lens).cpu().double()
    values = fo.unpack(v, block, d, True)
    ids = table.cpu().long()
    for b, t in enumerate(best.tolist()):
        want = values[ids[b, t // block], 0, t % block]
        assert float(((out[b] - want).abs() - HALF_STEP[dtype] * want.abs()).max()) <= 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("shift", [40, 100, 112, 118, 121, 124])
def test_tiny_queries_and_large_keys(d, shift):
    """Queries down to 2^-127 and keys up to 2^126: powers of two, by which neither a term nor a product is off."""
    q, k, v, table, lens = _inputs(EDGES, 8, 2, d, 16, BF, spread=1)
    gen = torch.Generator().manual_seed(shift)
    q.copy_(torch.randint(-31, 32, q.shape, generator=gen) / 8)
    want = fd.paged_decode_attention_fp4(q, k, v, table, lens)
    _check(want, q, k, v, table, lens, 16)
    k[:, :, 16 * d // 2 :] += shift
    assert torch.equal(fd.paged_decode_attention_fp4(q * 2.0**-shift, k, v, table, lens), want)
