"""GPU parity of the bounded-cache operators against their plain 64-bit forms (tests/bounded_oracle.py).

Tolerances, by arithmetic.  Let u be half a step of the tensors' type, relative to a value (bf16 2^-8, fp16 2^-11),
e = 2^-24 that of fp32, x a token's score times log2 e, and d a bound on the error of x.

* d: a dot product of D terms, each exact in fp32 (16-bit factors), summed in fp32 in any order, is off by at most
  (D - 1) e sum |q k|; the scale's rounding and product add 3 e |x|.  So d <= (D + 2) e scale log2(e) max sum |q k|.
* A probability 2^(x - M) / L is off, relatively, by 2 d ln 2 (itself and L) and by what the arithmetic adds: the
  exponentials' arguments |x - M| < 2^8 (beyond, the result is below every tolerance) are rounded by e 2^8 = 2^-16 at
  each of the at most three levels (unit, chunk, join), v_exp_f32, v_log_f32 and v_rcp_f32 by 2^-22 each, and the sums
  of n <= 2^15 positive terms, at most 2^8 of them one after the other in one accumulator, by 2^-16: 2^-13 in all.
* out = sum p v: the probabilities enter the product rounded to the type (u), the result leaves rounded (u): with
  A = sum p |v|, |error| <= (u + 2 d + 2^-13) A + u |out|, plus one smallest step for values near zero.
* The weights' sum over G heads has the same relative error without u; adding it to the table rounds by e |score|,
  on each call: n calls on weights of one sign by at most n e |last score|.
"""

import math
import threading
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from tests import bounded_oracle as ob
from tests.helpers import make_paged_inputs

pytestmark = pytest.mark.gpu

E = 2.0**-24
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
SMALLEST = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24}
EDGES = [700, 3, 0, 129, 2000, 64, 31, 1, 33, 32, 95, 511]


def _spread(q, k, table, lens, scale, kv_layout="token_major"):
    """d of the module's text: the largest sum |q k| over the batch's tokens."""
    k = ob.token_major(k.detach().cpu(), kv_layout).double().nan_to_num(0, 0, 0).abs()
    most = k.amax(dim=(0, 2)).amax(dim=0)  # per dim
    total = float((q.detach().cpu().double().abs() * most).sum(dim=2).max())
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else abs(scale)
    return (q.shape[2] + 2) * E * scale * math.log2(math.e) * total


def _check_out(out, q, k, v, table, lens, window=None, sinks=0, scale=None, kv_layout="token_major"):
    want, weights = ob.attend(q, k, v, table, lens, window, sinks, scale, kv_layout)
    size, _ = ob.attend(q, k, v.abs(), table, lens, window, sinks, scale, kv_layout)
    u, d = HALF_STEP[q.dtype], _spread(q, k, table, lens, scale, kv_layout)
    got = out.detach().cpu().double()
    bound = (u + 2 * d + 2.0**-13) * size + u * want.abs() + SMALLEST[q.dtype]
    assert bool(torch.isfinite(got).all())
    worst = ((got - want).abs() - bound).max()
    assert float(worst) <= 0, f"off by {float((got - want).abs().max()):.3g}, over the bound by {float(worst):.3g}"
    return weights, 2 * d + 2.0**-13


def _check_weights(scores, before, weights, rel, calls=1):
    want = before.detach().cpu().double() + weights
    got = scores.detach().cpu().double()
    bound = rel * weights + calls * E * want.abs() + 2.0**-120  # (weights below 2^-126 may be flushed)
    worst = ((got - want).abs() - bound).max()
    assert float(worst) <= 0, f"over the bound by {float(worst):.3g}"
    untouched = weights == 0
    assert torch.equal(scores.detach().cpu()[untouched], before.detach().cpu()[untouched])


def _poison(k, v, table, lens, block, window=None, sinks=0):
    """Fills every cached place that no row attends with NaN or an infinity."""
    seen = torch.zeros(k.shape[0], block, dtype=torch.bool)
    for b, n in enumerate(lens.tolist()):
        for t in ob.attended(min(max(n, 0), table.shape[1] * block), window, sinks):
            if 0 <= int(table[b, t // block]) < k.shape[0]:
                seen[int(table[b, t // block]), t % block] = True
    hidden = ~seen.to(k.device)
    bad = torch.tensor([math.nan, math.inf, -math.inf, math.nan], device=k.device, dtype=k.dtype)
    fill = bad.repeat(k.shape[3] // 4)
    for cache in (k, v):
        cache.copy_(torch.where(hidden[:, None, :, None], fill, cache))


HEADS = [(16, 2, 128), (32, 8, 128), (4, 4, 128), (16, 1, 128), (14, 2, 64), (40, 2, 64), (71, 1, 64), (34, 2, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize(("hq", "hkv", "d"), HEADS)
def test_window(dtype, block, hq, hkv, d):
    import flashdec_amd as fd

    q, k, v, table, lens = make_paged_inputs(EDGES, hq, hkv, d, block, dtype=dtype, seed=block + hq)
    for window, sinks in ((1, 0), (100, 5), (333, 64), (64, 0)):
        table2 = table.clone()
        for b, n in enumerate(EDGES):  # blocks that no longer hold an attended token belong to others
            table2[b, -(-sinks // block):max(0, n - window) // block] = -7 if b % 2 else 1 << 30
        k2, v2 = k.clone(), v.clone()
        _poison(k2, v2, table2, lens, block, window, sinks)
        out = fd.paged_decode_attention_window(q, k2, v2, table2, lens, window, sink_tokens=sinks)
        assert out.dtype == dtype
        _check_out(out, q, k, v, table2, lens, window, sinks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize(("hq", "hkv", "d"), HEADS)
def test_scored(dtype, block, hq, hkv, d):
    import flashdec_amd as fd

    q, k, v, table, lens = make_paged_inputs(EDGES, hq, hkv, d, block, dtype=dtype, seed=block + hq)
    _poison(k, v, table, lens, block)
    before = torch.rand(len(EDGES), hkv, table.shape[1] * block, device="cuda")
    scores = before.clone()
    out = fd.paged_decode_attention_scored(q, k, v, table, lens, scores)
    weights, rel = _check_out(out, q, k, v, table, lens)
    _check_weights(scores, before, weights, rel)
    again, twice = torch.empty_like(out), before.clone()
    fd.paged_decode_attention_scored_into(q, k, v, table, lens, again, twice)
    assert torch.equal(again, out) and torch.equal(twice, scores)  # the same bits
    fd.paged_decode_attention_scored(q, k, v, table, lens, scores)
    _check_weights(scores, before, 2 * weights, rel, calls=2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize(("hq", "hkv", "d"), HEADS)
def test_dim_major(dtype, block, hq, hkv, d):
    import flashdec_amd as fd

    q, k, v, table, lens = make_paged_inputs(EDGES, hq, hkv, d, block, dtype=dtype, seed=block + hq)
    for window, sinks in ((1, 0), (100, 5), (333, 64), (64, 0)):
        table2 = table.clone()
        for b, n in enumerate(EDGES):
            table2[b, -(-sinks // block):max(0, n - window) // block] = -7 if b % 2 else 1 << 30
        k2, v2 = k.clone(), v.clone()
        _poison(k2, v2, table2, lens, block, window, sinks)
        k2, v2 = (t.transpose(2, 3).contiguous() for t in (k2, v2))
        out = fd.paged_decode_attention_window(q, k2, v2, table2, lens, window, sinks, kv_layout="dim_major")
        _check_out(out, q, k, v, table2, lens, window, sinks)
    table[4, 3], table[9, 0] = -1, k.shape[0]  # (of 2000 and 32 tokens)
    k2, v2 = k.clone(), v.clone()
    _poison(k2, v2, table, lens, block)
    k2, v2 = (t.transpose(2, 3).contiguous() for t in (k2, v2))
    for kv_reuse in (False, True):
        before = torch.rand(len(EDGES), hkv, table.shape[1] * block, device="cuda")
        scores = before.clone()
        out = fd.paged_decode_attention_scored(q, k2, v2, table, lens, scores, kv_layout="dim_major", kv_reuse=kv_reuse)
        weights, rel = _check_out(out, q, k, v, table, lens)
        _check_weights(scores, before, weights, rel)


@pytest.mark.parametrize("layout", ["token_major", "dim_major"])
@pytest.mark.parametrize("heads", [(300, 1, 64), (256, 1, 128), (17, 1, 128)])
def test_wide_groups(heads, layout):
    import flashdec_amd as fd

    q, k, v, table, lens = make_paged_inputs([70, 0, 700, 33], *heads, 16, seed=5)
    kc, vc = (k, v) if layout == "token_major" else (t.transpose(2, 3).contiguous() for t in (k, v))
    _check_out(fd.paged_decode_attention_window(q, kc, vc, table, lens, 50, 20, kv_layout=layout), q, k, v, table, lens, 50, 20)
    before = torch.rand(4, heads[1], table.shape[1] * 16, device="cuda")
    scores = before.clone()
    out = fd.paged_decode_attention_scored(q, kc, vc, table, lens, scores, kv_layout=layout)
    weights, rel = _check_out(out, q, k, v, table, lens)
    _check_weights(scores, before, weights, rel)


# one row long enough for several chunks and joins' passes, one that ends inside a chunk, one short
@pytest.mark.parametrize(("lens", "heads"), [([20000, 5, 9000], (16, 2, 128)), ([33000], (8, 1, 64)),
                                             ([1], (2, 1, 128)), ([65], (2, 2, 64)), ([300] * 70, (8, 4, 128))])
def test_long_short_and_many_rows(lens, heads):
    import flashdec_amd as fd

    q, k, v, table, sl = make_paged_inputs(lens, *heads, 32, seed=9)
    before = torch.zeros(len(lens), heads[1], table.shape[1] * 32, device="cuda")
    scores = before.clone()
    out = fd.paged_decode_attention_scored(2 * q, k, v, table, sl, scores)
    weights, rel = _check_out(out, 2 * q, k, v, table, sl)
    _check_weights(scores, before, weights, rel)
    total = scores.double().sum(dim=2).cpu()
    assert torch.allclose(total, torch.full_like(total, heads[0] // heads[1]), rtol=rel + 2.0**-16)
    for window, sinks in ((4096, 4), (10**12, 0), (7, 10**12), (2500, 100)):
        _check_out(fd.paged_decode_attention_window(q, k, v, table, sl, window, sinks), q, k, v, table, sl, window, sinks)


SHORT = [320, 0, 1, 15, 16, 17, 31, 32, 33, 64, 127, 129, 255, 257, 300, 319]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize(("hq", "hkv", "d"), HEADS)
def test_scored_short_tables(dtype, block, hq, hkv, d):
    """Tables of ten tiles: a row is one workgroup's (not so in groups above 16 heads)."""
    import flashdec_amd as fd

    q, k, v, table, lens = make_paged_inputs(SHORT, hq, hkv, d, block, dtype=dtype, seed=block + hq)
    _poison(k, v, table, lens, block)
    before = torch.rand(len(SHORT), hkv, table.shape[1] * block, device="cuda")
    scores = before.clone()
    out = fd.paged_decode_attention_scored(q, k, v, table, lens, scores)
    weights, rel = _check_out(out, q, k, v, table, lens)
    _check_weights(scores, before, weights, rel)
    # the last block gone, lengths below zero and past the table
    table[0, -1], table[13, 0] = -1, k.shape[0]
    lens[4], lens[14] = -1, 2**31 - 1
    scores = before.clone()
    out = fd.paged_decode_attention_scored(q, k, v, table.long(), lens.long(), scores, sm_scale=-0.2, kv_reuse=True)
    dims = before.clone()
    other = fd.paged_decode_attention_scored(q, k.transpose(2, 3).contiguous(), v.transpose(2, 3).contiguous(), table, lens,
                                             dims, sm_scale=-0.2, kv_layout="dim_major")
    # (slots of row 14's table past its 300 tokens hold what was put there, so it has to be read as it stands)
    keep = torch.arange(len(SHORT)) != 14
    got, want = out[keep], (q[keep], k, v, table[keep], lens[keep])
    weights, rel = _check_out(got, *want, scale=-0.2)
    _check_weights(scores[keep], before[keep], weights, rel)
    weights, rel = _check_out(other[keep], *want, scale=-0.2)
    _check_weights(dims[keep], before[keep], weights, rel)


@pytest.mark.parametrize("layout", ["token_major", "dim_major"])
@pytest.mark.parametrize(("batch", "heads", "block", "tokens"), [
    (25, (32, 8, 128), 16, 1000), (25, (32, 8, 128), 32, 9568), (25, (32, 8, 128), 32, 9600), (192, (16, 1, 128), 8, 1984),
    (192, (16, 1, 64), 16, 2016), (100, (14, 2, 64), 32, 700), (32, (8, 8, 64), 16, 5000), (200, (34, 2, 128), 16, 90), (200, (71, 1, 64), 16, 5000),
    (300, (16, 2, 128), 16, 600), (256, (16, 1, 128), 32, 900)])
def test_scored_many_rows(batch, heads, block, tokens, layout):
    """Enough rows for one workgroup each, up to the longest whose scores fit LDS (9568, 1984 tokens) and past it, in
    lengths spread over all that a table may hold; said to be ragged, they are cut in chunks, and a pair's weights are
    added by a few workgroups in turn."""
    import flashdec_amd as fd

    lens = [max(0, (tokens * i * i) // ((batch - 1) ** 2)) for i in range(batch)]
    q, k, v, table, sl = make_paged_inputs(lens, *heads, block, seed=31)
    kc, vc = (k, v) if layout == "token_major" else (t.transpose(2, 3).contiguous() for t in (k, v))
    before = torch.rand(batch, heads[1], table.shape[1] * block, device="cuda")
    results = []
    for ragged in (False, True):
        scores = before.clone()
        out = fd.paged_decode_attention_scored(q, kc, vc, table, sl, scores, kv_layout=layout, ragged=ragged)
        results.append((out, scores))
    at = [0, 1, 2, batch // 3, batch // 2, batch - 2, batch - 1]
    for out, scores in results:
        weights, rel = _check_out(out[at], q[at], k, v, table[at], sl[at])
        _check_weights(scores[at], before[at], weights, rel)
    for window, sinks in ((1500, 40), (100, 0)):
        out = fd.paged_decode_attention_window(q, kc, vc, table, sl, window, sinks, kv_layout=layout)
        _check_out(out[at], q[at], k, v, table[at], sl[at], window, sinks)
        assert not bool(out[sl == 0].any())
    # every row, of both: each within its bound of the same exact result (values below 6 in magnitude, sums of
    # probabilities 1; weights up to the group's size, known up to d itself: 2.01 for 2)
    (a, sa), (b, sb) = results
    d = 2 * _spread(q, k, table, sl, None) + 2.0**-13
    assert float((a.float() - b.float()).abs().max()) <= 2 * (2 * HALF_STEP[q.dtype] + d) * float(v.float().abs().max())
    assert bool(((sa - sb).abs() <= 2.01 * (d * (sa - before).abs() + E * (1 + sa.abs())) + 2.0**-120).all())


def test_more_rows_than_a_grid_dimension_holds():
    import flashdec_amd as fd

    rows, at = 65600, [0, 1, 17, 65535, 65536, 65599]
    q, k, v, table, lens = make_paged_inputs([i % 41 for i in range(rows)], 2, 1, 64, 16, seed=6)
    out = fd.paged_decode_attention_window(q, k, v, table, lens, 7, 2)
    _check_out(out[at], q[at], k, v, table[at], lens[at], 7, 2)
    before = torch.rand(rows, 1, table.shape[1] * 16, device="cuda")
    scores = before.clone()
    out = fd.paged_decode_attention_scored(q, k, v, table, lens, scores)
    weights, rel = _check_out(out[at], q[at], k, v, table[at], lens[at])
    _check_weights(scores[at], before[at], weights, rel)
    total = (scores.double() - before.double()).sum(dim=2)[:, 0].cpu()
    assert torch.allclose(total, 2.0 * (lens.cpu() > 0).double(), atol=41 * 2 * (rel + 2 * E))
    want = ob.evict(k, v, table[at], lens[at], scores[at], 20, 2, 5)
    kept, new_lens = fd.paged_kv_evict(k, v, table, lens, scores, 20, 2, 5)
    assert torch.equal(kept[at].cpu(), want[0]) and torch.equal(new_lens.cpu(), lens.cpu().clamp(max=20))
    assert torch.equal(scores[at].cpu(), want[2])
    for cache, moved in ((k, want[3]), (v, want[4])):
        for b in at:
            for t in range(int(new_lens[b])):
                blk = int(table[b, t // 16])
                assert torch.equal(cache[blk, :, t % 16].cpu(), moved[blk, :, t % 16])


@pytest.mark.parametrize("layout", ["token_major", "dim_major"])
@pytest.mark.parametrize("block", [8, 32])
def test_pools_past_32_bits(block, layout):
    """Blocks more than 2^32 elements into the cache: the bits of the same rows in a small pool."""
    import flashdec_amd as fd

    lens, d, hkv = [700, 65, 300], 128, 2
    q, k, v, table, sl = make_paged_inputs(lens, 16, hkv, d, block, seed=8, kv_layout=layout)
    blocks = 2**32 // (hkv * block * d) + k.shape[0]
    far = blocks - k.shape[0]
    big_k, big_v = (torch.empty(blocks, *k.shape[1:], device="cuda", dtype=q.dtype) for _ in range(2))
    table2 = torch.where(table >= 0, table + far, table)
    big_k[far:].copy_(k)
    big_v[far:].copy_(v)
    assert torch.equal(fd.paged_decode_attention_window(q, big_k, big_v, table2, sl, 100, 5, kv_layout=layout),
                       fd.paged_decode_attention_window(q, k, v, table, sl, 100, 5, kv_layout=layout))
    for rows in (slice(0, 3), slice(1, 2)):  # in chunks, and whole
        cut = -(-max(lens[rows]) // block)
        one, two = (torch.zeros(len(lens[rows]), hkv, cut * block, device="cuda") for _ in range(2))
        assert torch.equal(
            fd.paged_decode_attention_scored(q[rows], big_k, big_v, table2[rows, :cut], sl[rows], one, kv_layout=layout),
            fd.paged_decode_attention_scored(q[rows], k, v, table[rows, :cut], sl[rows], two, kv_layout=layout))
        assert torch.equal(one, two)
    scores = torch.rand(3, hkv, table.shape[1] * block, device="cuda")
    small_k, small_v = k.clone(), v.clone()
    kept, new = fd.paged_kv_evict(big_k, big_v, table2, sl, scores.clone(), 64, 4, 20, kv_layout=layout)
    kept2, new2 = fd.paged_kv_evict(small_k, small_v, table, sl, scores, 64, 4, 20, kv_layout=layout)
    assert torch.equal(kept, kept2) and torch.equal(new, new2)
    assert torch.equal(big_k[far:], small_k) and torch.equal(big_v[far:], small_v)


def test_window_of_everything_is_decode():
    import flashdec_amd as fd

    q, k, v, table, lens = make_paged_inputs(EDGES, 16, 2, 128, 32, seed=4)
    for window, sinks in ((4000, 0), (1, 4000), (1000, 1000)):
        _check_out(fd.paged_decode_attention_window(q, k, v, table, lens, window, sinks), q, k, v, table, lens)


@pytest.mark.parametrize("op", ["window", "scored"])
def test_extreme_scores(op):
    """Scores far apart: a peak that takes all the weight, one that comes last, and scales of both signs."""
    import flashdec_amd as fd

    q, k, v, table, lens = make_paged_inputs([900, 640, 70], 16, 2, 128, 16, seed=6)
    k[table[0, 55].long(), :, 9] = q[0, ::8] * 3  # token 889 of row 0, next to the heads' own direction
    for scale in (None, 0.0, -0.25, 1.5):
        if op == "window":
            out = fd.paged_decode_attention_window(q, k, v, table, lens, 600, 4, sm_scale=scale)
            _check_out(out, q, k, v, table, lens, 600, 4, scale)
        else:
            before = torch.zeros(3, 2, table.shape[1] * 16, device="cuda")
            scores = before.clone()
            out = fd.paged_decode_attention_scored(q, k, v, table, lens, scores, sm_scale=scale)
            weights, rel = _check_out(out, q, k, v, table, lens, scale=scale)
            _check_weights(scores, before, weights, rel)


def _off_by_one(t):
    """The same values one element past an aligned place."""
    flat = torch.empty(t.numel() + 1, device=t.device, dtype=t.dtype)[1:]
    return flat.view(t.shape).copy_(t)


def _views(kind, q, k, v):
    """(q, k, v, kv_layout) with the same values in another memory layout."""
    if kind == "dim_major":
        return q, k.transpose(2, 3).contiguous(), v.transpose(2, 3).contiguous(), "dim_major"
    if kind == "dim_strided":
        return q, torch.stack((k, v), dim=4)[..., 0], torch.stack((v, k), dim=4)[..., 0], "token_major"
    if kind == "planes":  # [block, K/V, token, head, dim]
        both = torch.stack((k.transpose(1, 2), v.transpose(1, 2)), dim=1)
        return q, both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), "token_major"
    if kind == "odd_rows":  # rows of 130 elements: off the 16-byte lines
        wide = torch.zeros(*k.shape[:3], k.shape[3] + 2, device=k.device, dtype=k.dtype)
        wide2 = torch.zeros_like(wide)
        wide[..., :-2], wide2[..., :-2] = k, v
        return q, wide[..., :-2], wide2[..., :-2], "token_major"
    if kind == "unaligned":
        return q, _off_by_one(k), _off_by_one(v), "token_major"
    if kind == "unaligned_q":
        return _off_by_one(q), k, v, "token_major"
    return torch.stack((q, q), dim=3)[..., 0], k, v, "token_major"  # strided_q


LAYOUTS = ["dim_major", "dim_strided", "planes", "odd_rows", "unaligned", "unaligned_q", "strided_q"]


@pytest.mark.parametrize("kind", LAYOUTS)
@pytest.mark.parametrize(("hq", "hkv", "d"), [(16, 2, 128), (14, 2, 64), (40, 2, 64)])
def test_layouts(kind, hq, hkv, d):
    import flashdec_amd as fd

    q, k, v, table, lens = make_paged_inputs(EDGES, hq, hkv, d, 16, seed=12)
    q2, k2, v2, layout = _views(kind, q, k, v)
    out = fd.paged_decode_attention_window(q2, k2, v2, table, lens, 100, 5, kv_layout=layout)
    _check_out(out, q, k, v, table, lens, 100, 5)
    before = torch.rand(len(EDGES), hkv, table.shape[1] * 16, device="cuda")
    scores = before.clone()
    out = fd.paged_decode_attention_scored(q2, k2, v2, table, lens, scores, kv_layout=layout)
    weights, rel = _check_out(out, q, k, v, table, lens)
    _check_weights(scores, before, weights, rel)


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_strided_tables_lengths_outputs_and_scores(wide):
    import flashdec_amd as fd

    q, k, v, table, lens = make_paged_inputs(EDGES, 16, 2, 128, 16, seed=13)
    rows = len(EDGES)
    table2 = torch.full((table.shape[1] + 3, rows + 2), -1, device="cuda", dtype=wide)[2:-1, 1:-1].t()
    table2.copy_(table)
    lens2 = torch.stack((lens, -lens), dim=1).to(wide)[:, 0]
    out = torch.zeros(16, rows, 300, device="cuda", dtype=q.dtype)[..., 3:259:2].transpose(0, 1)
    assert fd.paged_decode_attention_window_into(q, k, v, table2, lens2, out, 100, 5) is out
    _check_out(out, q, k, v, table, lens, 100, 5)
    room = torch.rand(2, rows + 1, table.shape[1] * 16 + 7, device="cuda")
    old = room.clone()
    scores = room[:, 1:, 3:-4].transpose(0, 1)
    before = scores.clone()
    fd.paged_decode_attention_scored_into(q, k, v, table2, lens2, out, scores)
    weights, rel = _check_out(out, q, k, v, table, lens)
    _check_weights(scores, before, weights, rel)
    for part in (slice(None), 0), (slice(None), slice(None), slice(0, 3)), (slice(None), slice(None), slice(-4, None)):
        assert torch.equal(room[part], old[part])


@pytest.mark.parametrize(("hq", "hkv", "d"), [(16, 2, 128), (14, 2, 64), (40, 2, 64)])
def test_outputs_off_the_lines(hq, hkv, d):
    """Rows of unit stride at any element, of calls with one launch and with two."""
    import flashdec_amd as fd

    for lens, window in (([300, 5, 33], 40), ([300, 5, 33], 1000), ([2000, 5, 700], 1900)):
        q, k, v, table, sl = make_paged_inputs(lens, hq, hkv, d, 16, seed=14)
        room = torch.full((3, hq, d + 3), 7.0, device="cuda", dtype=q.dtype)
        out, far = _off_by_one(torch.empty_like(q)), room[..., 1:-2]
        for to in (out, far):
            _check_out(fd.paged_decode_attention_window_into(q, k, v, table, sl, to, window, 3), q, k, v, table, sl, window, 3)
            scores = torch.zeros(3, hkv, table.shape[1] * 16, device="cuda")
            _check_out(fd.paged_decode_attention_scored_into(q, k, v, table, sl, to, scores), q, k, v, table, sl)
        assert bool((room[..., 0] == 7).all()) and bool((room[..., -2:] == 7).all())


def test_rows_with_bad_blocks_negative_and_overlong_lengths():
    import flashdec_amd as fd

    q, k, v, table, _ = make_paged_inputs([320] * 6, 16, 2, 128, 32, seed=14)
    table[1, 2:4] = -1
    table[2, 9] = k.shape[0]
    table[3] = -1  # nothing left to attend
    lens = torch.tensor([320, 320, 320, 320, -5, 2**31 - 1], device="cuda", dtype=torch.int32)
    before = torch.rand(6, 2, 320, device="cuda")
    scores = before.clone()
    out = fd.paged_decode_attention_scored(q, k, v, table, lens, scores)
    weights, rel = _check_out(out, q, k, v, table, lens)
    _check_weights(scores, before, weights, rel)
    assert not bool(out[3:5].any())
    out = fd.paged_decode_attention_window(q, k, v, table, lens, 40, 33)
    _check_out(out, q, k, v, table, lens, 40, 33)
    assert not bool(out[3:5].any())


def test_shared_blocks_and_kv_reuse():
    import flashdec_amd as fd

    q, k, v, table, lens = make_paged_inputs([300, 400, 500], 16, 2, 128, 16, seed=15)
    table[1:, :8] = table[0, :8]
    plain = fd.paged_decode_attention_window(q, k, v, table, lens, 200, 100)
    _check_out(plain, q, k, v, table, lens, 200, 100)
    assert torch.equal(fd.paged_decode_attention_window(q, k, v, table, lens, 200, 100, kv_reuse=True), plain)
    one, two = (torch.zeros(3, 2, table.shape[1] * 16, device="cuda") for _ in range(2))
    plain = fd.paged_decode_attention_scored(q, k, v, table, lens, one)
    assert torch.equal(fd.paged_decode_attention_scored(q, k, v, table, lens, two, kv_reuse=True), plain)
    assert torch.equal(one, two)


# ------------------------------------------------------------------ eviction --
def _evict_case(lens, hkv, d, block, dtype=torch.bfloat16, seed=0, kv_layout="token_major"):
    _, k, v, table, sl = make_paged_inputs(lens, hkv, hkv, d, block, dtype=dtype, seed=seed, kv_layout=kv_layout)
    gen = torch.Generator().manual_seed(seed)
    scores = torch.randn((len(lens), hkv, table.shape[1] * block), generator=gen).mul_(1.5).exp_()
    scores[torch.rand(scores.shape, generator=gen) < 0.2] = 0.0
    return k, v, table, sl, scores.cuda()


def _check_evict(k, v, table, lens, scores, keep, sinks, recent, in_place, kv_layout="token_major"):
    import flashdec_amd as fd

    want = ob.evict(k, v, table, lens, scores, keep, sinks, recent, kv_layout)
    old_lens, old_scores = lens.clone(), scores.clone()
    if in_place:
        kept, new_lens = fd.paged_kv_evict(k, v, table, lens, scores, keep, sinks, recent, kv_layout=kv_layout)
        target = scores
    else:
        target = scores.clone()
        kept = torch.full((*scores.shape[:2], keep), 77, device="cuda", dtype=torch.int32)
        new_lens = torch.full_like(lens, 77)
        fd.paged_kv_evict_into(k, v, table, lens, scores, keep, kept, new_lens, sinks, recent, target,
                               kv_layout=kv_layout)
        assert torch.equal(scores.nan_to_num(7.5), old_scores.nan_to_num(7.5))
    assert torch.equal(lens, old_lens) and new_lens.dtype == lens.dtype
    assert torch.equal(new_lens.cpu().long(), want[1])
    assert torch.equal(kept.cpu(), want[0])
    assert torch.equal(target.cpu().view(torch.int32), want[2].view(torch.int32))
    for got, ref in ((k, want[3]), (v, want[4])):
        assert torch.equal(got.contiguous().view(torch.int16).cpu(), ref.contiguous().view(torch.int16))
    return kept, new_lens


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize(("block", "hkv", "d", "dtype"), [(8, 2, 128, torch.bfloat16), (16, 3, 64, torch.float16),
                                                          (32, 8, 128, torch.float16), (32, 1, 64, torch.bfloat16)])
@pytest.mark.parametrize(("keep", "sinks", "recent"), [(64, 4, 16), (1, 0, 0), (1, 1, 0), (33, 13, 20), (700, 0, 100),
                                                       (1999, 37, 1), (5000, 4, 64)])
def test_evict(block, hkv, d, dtype, keep, sinks, recent, in_place):
    case = _evict_case(EDGES, hkv, d, block, dtype, seed=block + keep)
    _check_evict(*case, keep, sinks, recent, in_place)


@pytest.mark.parametrize("lens", [[20000, 5, 4097], [33001], [256] * 70, [16000, 4097, 700], [70001]])
@pytest.mark.parametrize("share", [0.1, 0.5, 0.95])
def test_evict_long_and_many_rows(lens, share):
    case = _evict_case(lens, 2, 64, 32, seed=len(lens))
    _check_evict(*case, max(80, int(max(lens) * share)), 4, 64, True)


@pytest.mark.parametrize("kind", ["zeros", "equal", "nan", "infinite", "negative", "two", "denormal"])
def test_evict_order_of_scores(kind):
    k, v, table, lens, scores = _evict_case([1000, 333], 2, 64, 16, seed=5)
    gen = torch.Generator().manual_seed(3)
    pick = torch.rand(scores.shape, generator=gen).cuda()
    if kind == "zeros":
        scores.zero_()
        scores[pick < 0.5] = -0.0
    elif kind == "equal":
        scores.fill_(0.37)
    elif kind == "nan":
        scores[pick < 0.7] = math.nan
        scores[pick < 0.2] = -math.nan
        scores[(pick > 0.75) & (pick < 0.8)] = -math.inf
    elif kind == "infinite":
        scores[pick < 0.3] = math.inf
        scores[pick > 0.6] = -math.inf
    elif kind == "negative":
        scores.sub_(1.0)
    elif kind == "two":
        scores.copy_((pick < 0.4).float() + 1.0)
    else:
        scores.copy_(torch.randint(0, 9, scores.shape, generator=gen).int().cuda().view(torch.float32))
    for keep in (200, 400):
        _check_evict(k.clone(), v.clone(), table, lens, scores.clone(), keep, 3, 20, True)


@pytest.mark.parametrize("kind", ["dim_major", "dim_strided", "planes", "odd_rows", "unaligned"])
@pytest.mark.parametrize("d", [64, 128])
def test_evict_layouts(kind, d):
    k, v, table, lens, scores = _evict_case([700, 3, 0, 300], 2, d, 16, seed=8)
    _, k2, v2, layout = _views(kind, k[:, :, 0], k, v)
    _check_evict(k2, v2, table, lens, scores, 100, 4, 30, True, layout)


@pytest.mark.parametrize("block", [8, 16, 32])
@pytest.mark.parametrize(("hkv", "d", "dtype"), [(2, 128, torch.bfloat16), (3, 64, torch.float16)])
@pytest.mark.parametrize(("keep", "sinks", "recent"), [(64, 4, 16), (1, 0, 0), (33, 13, 20), (700, 0, 100), (129, 9, 64)])
def test_evict_dim_major(block, hkv, d, dtype, keep, sinks, recent):
    case = _evict_case(EDGES, hkv, d, block, dtype, seed=keep, kv_layout="dim_major")
    _check_evict(*case, keep, sinks, recent, True, kv_layout="dim_major")


def test_evict_dim_major_bad_blocks_and_long_rows():
    k, v, table, lens, scores = _evict_case([9000, 700, 320, 400], 2, 128, 32, seed=3, kv_layout="dim_major")
    table[1, 2:4], table[2, 9], table[3] = -1, k.shape[0], -1
    _check_evict(k, v, table, lens, scores, 300, 4, 30, True, kv_layout="dim_major")


def test_evict_strided_tables_lengths_and_scores():
    k, v, table, lens, scores = _evict_case([700, 3, 0, 300], 2, 64, 16, seed=8)
    table2 = torch.full((table.shape[1] + 3, 6), -1, device="cuda", dtype=torch.int64)[2:-1, 1:-1].t()
    table2.copy_(table)
    lens2 = torch.stack((lens, -lens), dim=1).long()[:, 0]
    room = torch.rand(2, 5, scores.shape[2] + 7, device="cuda")
    view = room[:, 1:, 3:-4].transpose(0, 1)
    view.copy_(scores)
    _check_evict(k, v, table2, lens2, view, 100, 4, 30, True)


def test_evict_bad_blocks_negative_and_overlong_lengths():
    k, v, table, _, scores = _evict_case([320] * 5, 2, 128, 32, seed=3)
    table[1, 2:4] = -1
    table[2, 9] = k.shape[0]
    table[3] = -1
    lens = torch.tensor([320, 320, 2**31 - 1, 320, -4], device="cuda", dtype=torch.int32)
    _check_evict(k, v, table, lens, scores, 150, 4, 20, True)


def test_evict_leaves_a_shared_prefix_alone():
    k, v, table, lens, scores = _evict_case([300, 300, 250], 2, 128, 16, seed=4)
    table[1:, :4] = table[0, :4]
    _check_evict(k, v, table, lens, scores, 128, 64, 16, True)


# ------------------------------------------------------- together, graphs, streams --
def test_a_run_of_them_together():
    """Rows of unequal lengths generated past their budget twice: every step's attention is that over
    the tokens the plain eviction would have left, whatever order of calls came before."""
    import flashdec_amd as fd

    hq, hkv, d, block, steps, budget, keep = 8, 2, 64, 16, 60, 128, 96
    _, k, v, table, lens = make_paged_inputs([100, 61, 9], hq, hkv, d, block, seed=21, table_width=8, pool_factor=4)
    table.copy_(torch.randperm(k.shape[0], generator=torch.Generator().manual_seed(1))[:24].view(3, 8))
    assert k.shape[0] >= 24
    gen = torch.Generator().manual_seed(2)
    q, k_new, v_new = (torch.randn((steps, 3, h, d), generator=gen).to(torch.bfloat16).cuda() for h in (hq, hkv, hkv))
    scores = torch.zeros(3, hkv, 128, device="cuda")
    positions = lens.clone()
    for i in range(steps):
        rows = torch.arange(3, device="cuda")
        ids, off = table[rows, (lens // block).long()], lens % block
        q_rot = fd.fused_rope_kv_append(q[i], k_new[i], v_new[i], k, v, ids, off, positions)
        lens += 1
        positions += 1
        before = scores.clone()
        out = fd.paged_decode_attention_scored(q_rot, k, v, table, lens, scores)
        weights, rel = _check_out(out, q_rot, k, v, table, lens)
        _check_weights(scores, before, weights, rel)
        out = fd.paged_decode_attention_window(q_rot, k, v, table, lens, 40, 4)
        _check_out(out, q_rot, k, v, table, lens, 40, 4)
        if int(lens.max()) == budget:
            _, new = _check_evict(k, v, table, lens, scores, keep, 4, 20, True)
            lens.copy_(new)
    # (cut after steps 28 and 60; the second row has 89 tokens at the first cut, 121 at the second)
    assert lens.tolist() == [96, 96, 69] and positions.tolist() == [160, 121, 69]


@pytest.mark.parametrize("op", ["window", "scored"])
def test_captured_calls_own_their_workspace(op):
    """Two graphs captured on one stream, replayed in any order with eager calls of larger shapes between."""
    import flashdec_amd as fd

    def make(lens, seed):
        q, k, v, table, sl = make_paged_inputs(lens, 16, 2, 128, 32, seed=seed)
        scores = torch.zeros(len(lens), 2, table.shape[1] * 32, device="cuda")
        out = torch.empty_like(q)

        def call():
            if op == "window":
                fd.paged_decode_attention_window_into(q, k, v, table, sl, out, 900, 4)
            else:
                fd.paged_decode_attention_scored_into(q, k, v, table, sl, out, scores)

        return call, out, scores

    cases = [make([2000, 700, 64], 1), make([300, 1500], 2)]
    larger, _, _ = make([3000] * 6, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    wants, graphs = [], []
    with torch.cuda.stream(side):
        for call, out, scores in cases:
            call()
            wants.append((out.clone(), scores.clone()))
    torch.cuda.synchronize()
    for call, _, _ in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
        graphs.append(graph)
    for first in (0, 1, 0):
        for i in (first, 1 - first):
            _, out, scores = cases[i]
            out.zero_()
            scores.zero_()
            graphs[i].replay()
            with torch.cuda.stream(side):
                larger()
            torch.cuda.synchronize()
            assert torch.equal(out, wants[i][0]) and torch.equal(scores, wants[i][1])


def test_eviction_in_a_graph():
    """Scored decode and eviction captured once, replayed on new contents: the loop with no host in it."""
    import flashdec_amd as fd

    k0, v0, table, lens, scores0 = _evict_case([500, 90, 300], 2, 128, 16, seed=6)
    k, v, scores = k0.clone(), v0.clone(), scores0.clone()
    q = torch.randn(3, 16, 128, device="cuda").to(torch.bfloat16)
    out = torch.empty_like(q)
    kept, new_lens = torch.empty(3, 2, 128, device="cuda", dtype=torch.int32), torch.empty_like(lens)

    def step():
        fd.paged_decode_attention_scored_into(q, k, v, table, lens, out, scores)
        fd.paged_kv_evict_into(k, v, table, lens, scores, 128, kept, new_lens, 4, 32)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(4):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)))
        results = []
        for run in (graph.replay, step):
            k.copy_(k0), v.copy_(v0), scores.copy_(scores0)
            run()
            torch.cuda.synchronize()
            results.append([t.clone() for t in (out, scores, kept, new_lens, k, v)])
        for a, b in zip(*results):
            assert torch.equal(a, b)


def test_threads_and_streams_share_nothing():
    import flashdec_amd as fd

    cases = []
    for i in range(4):
        q, k, v, table, lens = make_paged_inputs([1500 + 100 * i, 40, 700], 16, 2, 128, 32, seed=i)
        want = fd.paged_decode_attention_window(q, k, v, table, lens, 1000, 4)
        scores = torch.zeros(3, 2, table.shape[1] * 32, device="cuda")
        both = fd.paged_decode_attention_scored(q, k, v, table, lens, scores)
        cases.append((q, k, v, table, lens, want, both, scores))
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        q, k, v, table, lens, want, both, table_want = cases[i]
        stream = torch.cuda.Stream() if i % 2 else torch.cuda.default_stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                scores = torch.zeros_like(table_want)
                a = fd.paged_decode_attention_window(q, k, v, table, lens, 1000, 4)
                b = fd.paged_decode_attention_scored(q, k, v, table, lens, scores)
                if not (torch.equal(a, want) and torch.equal(b, both) and torch.equal(scores, table_want)):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_the_kept_call_follows_its_arguments():
    """Alternating calls of the same shapes on other tensors, and of other settings on the same ones."""
    import flashdec_amd as fd

    a, b = (make_paged_inputs([600, 40], 16, 2, 128, 32, seed=s) for s in (1, 2))
    for _ in range(2):
        for case in (a, b):
            for window, sinks, scale in ((100, 4, None), (100, 5, None), (101, 5, 0.3)):
                out = fd.paged_decode_attention_window(*case, window, sinks, sm_scale=scale)
                _check_out(out, *case, window, sinks, scale)
            scores = torch.zeros(2, 2, 608, device="cuda")
            fd.paged_decode_attention_scored(*case, scores)
            _check_weights(scores, torch.zeros_like(scores), *_check_out(
                fd.paged_decode_attention_scored(*case, torch.zeros_like(scores)), *case))
    # an unaligned query of the same shape and strides takes another kernel
    q = _off_by_one(a[0])
    assert q.stride() == a[0].stride()
    _check_out(fd.paged_decode_attention_window(q, *a[1:], 101, 5, sm_scale=0.3), *a, 101, 5, 0.3)
    _check_out(fd.paged_decode_attention_window(*a, 101, 5, sm_scale=0.3), *a, 101, 5, 0.3)


def test_which_kernels_run():
    """From the library's launch record: the kernel that each rule's side takes."""
    import flashdec_amd as fd
    from flashdec_amd import _lib

    def mfma(mode, block=32, d=128, ncb=1, nt="true", dm="false"):
        return f"fd::bounded_mfma_kernel<__bf16, {block}, {d}, {ncb}, {mode}, 4, {nt}, {dm}>"

    def scored(lens, heads, block=32, **settings):
        q, k, v, table, sl = make_paged_inputs(lens, *heads, block, seed=3)
        fd.paged_decode_attention_scored(q, k, v, table, sl, torch.zeros(len(lens), heads[1], table.shape[1] * block,
                                                                         device="cuda"), **settings)
        return _lib.last_launch()

    def window(lens, heads, window, sinks, block=32, kind=None, **settings):
        q, k, v, table, sl = make_paged_inputs(lens, *heads, block, seed=3)
        if kind is not None:
            q, k, v, settings["kv_layout"] = _views(kind, q, k, v)
        fd.paged_decode_attention_window(q, k, v, table, sl, window, sinks, **settings)
        return _lib.last_launch()

    def evict(lens, hkv, d, keep, kind=None):
        k, v, table, sl, scores = _evict_case(lens, hkv, d, 16)
        layout = "token_major"
        if kind is not None:
            _, k, v, layout = _views(kind, k[0], k, v)
        fd.paged_kv_evict(k, v, table, sl, scores, keep, kv_layout=layout)
        return _lib.last_launch()

    whole, chunk, one = 2, 1, 0
    join = "fd::bounded_join_kernel<__bf16, 128, {}>"
    _lib.record_launches(True)
    try:
        # whole rows up to ten tiles, or with a row for three CUs of four, or one and a half rows a CU; else chunks
        assert scored([320, 5], (16, 2, 128)) == [mfma(whole)]
        assert scored([352, 5], (16, 2, 128)) == [mfma(chunk), join.format(8)]
        assert scored([700] * 24, (32, 8, 128), 16) == [mfma(whole, 16)]
        assert scored([700] * 24, (32, 8, 128), 16, ragged=True) == [mfma(chunk, 16), join.format(4)]
        assert scored([700] * 48, (32, 8, 128), 16) == [mfma(whole, 16)]
        assert scored([700] * 40, (32, 8, 128), 16) == [mfma(chunk, 16), join.format(4)]
        assert scored([700] * 23, (32, 8, 128), 16) == [mfma(chunk, 16), join.format(4)]
        assert scored([100], (34, 2, 128), kv_reuse=True) == [mfma(chunk, ncb=2, nt="false"), join.format(8)]
        # one chunk a row needs no join
        assert window([2000, 5], (16, 2, 128), 40, 4) == [mfma(one)]
        assert window([2000, 5], (16, 2, 128), 1500, 4) == [mfma(one), join.format(0)]
        assert window([300], (14, 2, 64), 50, 4, 8) == [mfma(one, 8, 64)]
        assert window([300], (40, 2, 64), 50, 4, kind="dim_major") == [mfma(one, d=64, dm="true")]
        assert window([2000], (16, 2, 128), 1500, 4, 8, "dim_major") == [mfma(one, 8, dm="true"), join.format(0)]
        for kind in ("dim_strided", "unaligned", "strided_q"):
            assert window([300], (16, 2, 128), 50, 4, kind=kind)[0] == "fd::bounded_generic_kernel<__bf16, 128, false>"
        # keys in registers for the longest row of the table, larger workgroups past one a CU
        assert evict([400, 90], 2, 128, 100) == ["fd::evict_select_kernel<4, true>", "fd::evict_move_kernel<128, 256>"]
        assert evict([400] * 70, 4, 64, 300) == ["fd::evict_select_kernel<4, true>", "fd::evict_move_kernel<64, 512>"]
        assert evict([10000], 1, 64, 300)[0] == "fd::evict_select_kernel<16, true>"
        assert evict([20000], 1, 64, 300)[0] == "fd::evict_select_kernel<32, true>"
        assert evict([33000], 1, 64, 300)[0] == "fd::evict_select_kernel<32, false>"
        assert evict([400], 1, 64, 300, "dim_major")[1] == "fd::evict_move_dm_kernel<64>"
        assert evict([400], 1, 64, 300, "unaligned")[1] == "fd::evict_move_generic_kernel"
    finally:
        _lib.record_launches(False)


def test_more_calls_than_are_kept():
    """Twenty shapes in turn, the workspaces of later ones larger: the same bits the second and third time."""
    import numpy as np

    import flashdec_amd as fd

    cases = [make_paged_inputs([400 + 90 * i, 40], 16, 2, 128, 32, seed=i) for i in range(20)]
    first = []
    for turn in range(3):
        for i, case in enumerate(cases):
            scores = torch.rand((2, 2, case[3].shape[1] * 32), generator=torch.Generator().manual_seed(i)).cuda()
            before = scores.clone()
            got = [fd.paged_decode_attention_window(*case, 900, 4), fd.paged_decode_attention_scored(*case, scores),
                   scores.clone(), *fd.paged_kv_evict(case[1].clone(), case[2].clone(), *case[3:], scores, 64, 4, 16), scores]
            if turn == 0:
                _check_out(got[0], *case, 900, 4)
                weights, rel = _check_out(got[1], *case)
                _check_weights(got[2], before, weights, rel)
                first.append(got)
            else:
                assert all(torch.equal(a, b) for a, b in zip(got, first[i]))
    # a setting that no table of calls can hold
    case, scale = cases[0], np.array(0.05)
    for _ in range(2):
        _check_out(fd.paged_decode_attention_window(*case, 900, 4, sm_scale=scale), *case, 900, 4, 0.05)


def test_refusals():
    import flashdec_amd as fd

    q, k, v, table, lens = make_paged_inputs([60, 40], 4, 2, 64, 16, seed=1)
    scores = torch.zeros(2, 2, 64, device="cuda")
    window = fd.paged_decode_attention_window
    for bad in (0, -3, 2.5, True, None, "7"):
        with pytest.raises(ValueError, match="window"):
            window(q, k, v, table, lens, bad)
    for bad in (-1, 0.5, False, None):
        with pytest.raises(ValueError, match="sink_tokens"):
            window(q, k, v, table, lens, 5, bad)
    with pytest.raises(ValueError, match="kv_layout"):
        window(q, k, v, table, lens, 5, kv_layout="rows")
    with pytest.raises(ValueError, match="same dtype"):
        window(q.half(), k, v, table, lens, 5)
    with pytest.raises(ValueError, match="same shape as q"):
        fd.paged_decode_attention_window_into(q, k, v, table, lens, q[:1].clone(), 5)
    with pytest.raises(ValueError, match="overlapping"):
        fd.paged_decode_attention_window_into(q, k, v, table, lens, q[:1].expand_as(q), 5)
    for bad in (scores[:1], scores[:, :, :63], scores.half(), scores.cpu(), scores[:1].expand(2, 2, 64)):
        with pytest.raises(ValueError, match="scores"):
            fd.paged_decode_attention_scored(q, k, v, table, lens, bad)
        with pytest.raises(ValueError):
            fd.paged_kv_evict(k, v, table, lens, bad, 20)
    for keep, sinks, recent in ((0, 0, 0), (20, 11, 10), (20, -1, 0), (20, 0, -1), (20.0, 0, 0), (True, 0, 0)):
        with pytest.raises(ValueError, match="keep|sink_tokens|recent_tokens"):
            fd.paged_kv_evict(k, v, table, lens, scores, keep, sinks, recent)
    with pytest.raises(ValueError, match="different tensors"):
        fd.paged_kv_evict(k, k, table, lens, scores, 20)
    with pytest.raises(ValueError, match="overlapping"):
        fd.paged_kv_evict(k[:1].expand_as(k), v, table, lens, scores, 20)
    kept, new = torch.empty(2, 2, 20, device="cuda", dtype=torch.int32), torch.empty_like(lens)
    for bad_kept, bad_new in ((kept.long(), new), (kept[:, :, :19], new), (kept.transpose(0, 1), new[:1]),
                              (kept, new.long()), (kept, lens)):
        with pytest.raises(ValueError):
            fd.paged_kv_evict_into(k, v, table, lens, scores, 20, bad_kept, bad_new)
    room = torch.zeros(2, 2, 65, device="cuda")
    with pytest.raises(ValueError, match="apart"):
        fd.paged_kv_evict_into(k, v, table, lens, room[:, :, :64], 20, kept, new, new_scores=room[:, :, 1:])


@pytest.mark.parametrize("kind", ["numpy", "tensor"])
def test_a_scale_changed_in_place(kind):
    """The scale's value at each call counts, whatever object holds it."""
    import numpy as np

    import flashdec_amd as fd

    q, k, v, table, lens = make_paged_inputs([600, 40], 16, 2, 128, 32, seed=9)
    scale = np.zeros(()) if kind == "numpy" else torch.zeros(())
    for value in (0.05, 0.3, -0.1, 0.05):
        scale[...] = value
        out = fd.paged_decode_attention_window(q, k, v, table, lens, 500, 4, sm_scale=scale)
        _check_out(out, q, k, v, table, lens, 500, 4, float(scale))
        before = torch.zeros(2, 2, 608, device="cuda")
        scores = before.clone()
        out = fd.paged_decode_attention_scored(q, k, v, table, lens, scores, sm_scale=scale)
        _check_weights(scores, before, *_check_out(out, q, k, v, table, lens, scale=float(scale)))


@pytest.mark.parametrize("kind", [None, "unaligned", "dim_major"])
@pytest.mark.parametrize(("lens", "heads"), [([300, 40, 64], (16, 2, 128)), ([2000, 700, 64], (16, 2, 128)),
                                             ([2000, 700, 64], (14, 2, 64)), ([300, 40, 64], (40, 2, 64))])
def test_rows_that_attend_nan(lens, heads, kind):
    """A NaN or an infinite score makes its head's whole row NaN, in the output and in the table, as the
    softmax's definition has it; the other rows keep their values."""
    import flashdec_amd as fd

    q, k, v, table, sl = make_paged_inputs(lens, *heads, 16, seed=31)
    k[table[0, 0].long(), 0, 3, 5] = math.nan  # row 0: token 3 of KV head 0
    k[table[1, 0].long(), 1, 2, 7] = math.inf  # row 1: token 2 of KV head 1, the heads whose query is positive there
    table[0, 1] = -1  # 16 tokens of row 0 that no head attends
    q2, k2, v2, layout = (q, k, v, "token_major") if kind is None else _views(kind, q, k, v)
    before = torch.rand(3, heads[1], table.shape[1] * 16, device="cuda")
    scores = before.clone()
    out = fd.paged_decode_attention_scored(q2, k2, v2, table, sl, scores, kv_layout=layout).cpu().double()
    want, weights = ob.attend(q, k, v, table, sl)
    assert bool(want[0].isnan().any()) and bool(want[1].isnan().any()) and not bool(want[2].isnan().any())
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(scores.cpu().isnan(), weights.isnan())
    # rows and heads without: as of inputs that hold neither
    k = k.nan_to_num(0, 0, 0)
    clean, rest = ob.attend(q, k, v, table, sl)
    size, _ = ob.attend(q, k, v.abs(), table, sl)
    u, d = HALF_STEP[q.dtype], _spread(q, k, table, sl, None)
    heads_of = want.isnan().view(3, heads[1], -1).any(dim=2)  # [row, KV head]
    group = heads[0] // heads[1]
    for b, h in (~heads_of).nonzero().tolist():
        rows = slice(h * group, (h + 1) * group)
        bound = (u + 2 * d + 2.0**-13) * size[b, rows] + u * clean[b, rows].abs() + SMALLEST[q.dtype]
        assert float(((out[b, rows] - clean[b, rows]).abs() - bound).max()) <= 0
        _check_weights(scores[b:b + 1, h:h + 1], before[b:b + 1, h:h + 1], rest[b:b + 1, h:h + 1], 2 * d + 2.0**-13)


def test_evictions_on_two_streams_at_once():
    """Evictions of the same shapes, on two streams in turn and on both at once: each has scratch of its own."""
    import flashdec_amd as fd

    cases = [_evict_case([5000, 90, 3000, 4000], 4, 128, 16, seed=s) for s in (1, 2)]
    wants = [ob.evict(k, v, table, lens, scores, 2500, 4, 100) for k, v, table, lens, scores in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(6):
        copies, got = [], []
        for k, v, table, lens, scores in cases:
            copies.append((k.clone(), v.clone(), table, lens, scores.clone()))
        torch.cuda.synchronize()
        for stream, case in zip(streams, copies):
            with torch.cuda.stream(stream):
                got.append(fd.paged_kv_evict(*case, 2500, 4, 100))
        torch.cuda.synchronize()
        for (k, v, _, _, scores), (kept, new), want in zip(copies, got, wants):
            assert torch.equal(kept.cpu(), want[0]) and torch.equal(new.cpu().long(), want[1])
            assert torch.equal(scores.cpu(), want[2]) and torch.equal(k.cpu(), want[3]) and torch.equal(v.cpu(), want[4])


def test_refusals_do_not_hang_on_earlier_calls():
    """A value that equals a valid one but is no integer is refused after the valid call too."""
    import numpy as np

    import flashdec_amd as fd

    q, k, v, table, lens = make_paged_inputs([60, 40], 4, 2, 64, 16, seed=1)
    k2, v2, scores = k.clone(), v.clone(), torch.rand(2, 2, 64, device="cuda")
    for _ in range(2):
        fd.paged_decode_attention_window(q, k, v, table, lens, 1, 1)
        fd.paged_kv_evict(k2, v2, table, lens, scores, 1, 0, 1)
    kept, new = torch.empty(2, 2, 1, device="cuda", dtype=torch.int32), torch.empty_like(lens)
    for bad in (True, 1.0, np.int64(1), np.array(1), np.ones(3), [1], torch.tensor(1)):
        with pytest.raises(ValueError, match="window"):
            fd.paged_decode_attention_window(q, k, v, table, lens, bad, 1)
        with pytest.raises(ValueError, match="sink_tokens"):
            fd.paged_decode_attention_window(q, k, v, table, lens, 1, bad)
        for keep, sinks, recent in ((bad, 0, 1), (1, bad, 0), (1, 0, bad)):
            with pytest.raises(ValueError, match="keep|sink_tokens|recent_tokens"):
                fd.paged_kv_evict_into(k2, v2, table, lens, scores, keep, kept, new, sinks, recent)


def test_threads_on_one_stream_share_nothing_and_all_finish():
    """Four threads at once, two on the default stream and two on their own: every iteration of each has the
    results of the call alone, and an error in a thread is one of the test."""
    import flashdec_amd as fd

    cases = []
    for i in range(4):
        q, k, v, table, lens = make_paged_inputs([1500 + 100 * i, 40, 700], 16, 2, 128, 32, seed=i)
        scores = torch.rand((3, 2, table.shape[1] * 32), generator=torch.Generator().manual_seed(i)).cuda()
        cases.append((q, k, v, table, lens, scores))
    together = threading.Barrier(4, timeout=60)

    def step(q, k, v, table, lens, scores):
        k, v, scores = k.clone(), v.clone(), scores.clone()
        window = fd.paged_decode_attention_window(q, k, v, table, lens, 1000, 4)
        scored = fd.paged_decode_attention_scored(q, k, v, table, lens, scores)
        kept, new_lens = fd.paged_kv_evict(k, v, table, lens, scores, 300, 4, 50)
        return window, scored, kept, new_lens, scores, k, v

    wants = [step(*case) for case in cases]
    torch.cuda.synchronize()

    def work(i):
        same = 0
        with torch.cuda.stream(torch.cuda.Stream() if i % 2 else torch.cuda.default_stream()):
            together.wait()
            for _ in range(20):
                same += all(torch.equal(got, want) for got, want in zip(step(*cases[i]), wants[i]))
        return same

    with ThreadPoolExecutor(4) as pool:
        running = [pool.submit(work, i) for i in range(4)]
        assert [job.result() for job in running] == [20] * 4
