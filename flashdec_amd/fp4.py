"""A paged cache held in 4 bits on MI355X through ``libflashdec_hip.so``.

A token's keys and values take 17/32 of a byte a dim instead of two bytes, so a
pool holds 3.8 times the tokens, and decode reads that much less (no counterpart
in the reference, whose caches are 16-bit).  32 neighbouring dims of a token's head
share a power of two and each is one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their
negatives times it (MX fp4); the power is the least that leaves the group's largest
at 7 or below.

* :func:`fp4_block_bytes`: bytes of one KV head's block.  The pools are uint8
  ``[num_blocks, num_kv_heads, fp4_block_bytes(block_size, head_dim)]``.
* :func:`fused_rope_kv_append_fp4` (and :func:`kv_append_fp4`, without rotation)
  quantise new tokens into their slots: a decode step's, or a prompt's.
* :func:`paged_decode_attention_fp4` attends it.
* :func:`paged_kv_read_fp4` gives the tokens of any slots back as 16-bit values.

A step of a batch::

    k_cache = torch.empty((num_blocks, num_kv_heads, fp4_block_bytes(32, 128)), device="cuda", dtype=torch.uint8)
    v_cache = torch.empty_like(k_cache)
    ...
    q_rot = fused_rope_kv_append_fp4(q, k, v, k_cache, v_cache, block_ids, block_offsets, positions)
    out = paged_decode_attention_fp4(q_rot, k_cache, v_cache, block_tables, seq_lens)  # lengths with the new tokens
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._fused_rope_kv_append import _check_cos_sin_table, _validate_index_values
from .bounded import _apart, _Call, _check_out, _keep, _kept, _launch, _number, _reach, _spread_out

_BLOCK_SIZES = (8, 16, 32)
_HEAD_DIMS = (64, 128)


def fp4_block_bytes(block_size, head_dim):
    """Bytes of one KV head's block of a 4-bit pool: the codes, then a scale byte for each 32 dims of a token."""
    if block_size not in _BLOCK_SIZES:
        raise ValueError("a 4-bit cache supports block_size 8, 16, or 32")
    if head_dim not in _HEAD_DIMS:
        raise ValueError("a 4-bit cache supports head_dim 64 or 128")
    return block_size * head_dim * 17 // 32


def _check_pools(k_cache, v_cache, head_dim, device):
    """The 4-bit pools' contract; returns the block size."""
    for name, pool in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not isinstance(pool, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not pool.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")
        if pool.device != device:
            raise ValueError("the caches and the other tensors must be on the same CUDA device")
        if pool.dtype != torch.uint8 or pool.dim() != 3:
            raise ValueError(f"{name} must be a uint8 tensor of shape [num_blocks, num_kv_heads, block_bytes]")
        if pool.shape[0] <= 0 or pool.shape[1] <= 0:
            raise ValueError("num_blocks and num_kv_heads must be positive")
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have the same shape")
    if head_dim not in _HEAD_DIMS:
        raise ValueError("a 4-bit cache supports head_dim 64 or 128")
    block_size = k_cache.shape[2] * 32 // (17 * head_dim)
    if block_size not in _BLOCK_SIZES or k_cache.shape[2] != fp4_block_bytes(block_size, head_dim):
        raise ValueError("a block of a 4-bit cache must hold fp4_block_bytes(block_size, head_dim) bytes")
    for name, pool in (("k_cache", k_cache), ("v_cache", v_cache)):
        if pool.stride(2) != 1 or pool.stride(0) % 16 or pool.stride(1) % 16 or pool.data_ptr() % 16:
            raise ValueError(f"{name}'s blocks must be contiguous and lie on 16-byte lines")
    return block_size


def _check_written(pools):
    if not all(_spread_out(pool) for pool in pools):
        raise ValueError("k_cache and v_cache must have no overlapping elements")


def _check_rows(name, t, tokens, heads, head_dim, dtype, device):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dim() != 3 or t.shape[0] != tokens or t.shape[2] != head_dim or (heads is not None and t.shape[1] != heads):
        raise ValueError("q, k, v and the outputs must have shape [tokens, heads, head_dim], of equal tokens and head_dim")
    if t.dtype != dtype:
        raise ValueError("q, k, v and q_out must have the same dtype")
    if t.device != device:
        raise ValueError("the caches and the other tensors must be on the same CUDA device")
    if t.stride(2) != 1:
        raise ValueError(f"{name} must have unit dim stride")


def _check_indices(tokens, device, **tensors):
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.dim() != 1 or t.shape[0] != tokens:
            raise ValueError(f"{name} must have one value per token")
        if t.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name} must be int32 or int64")
        if t.device != device:
            raise ValueError("the caches and the other tensors must be on the same CUDA device")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")


class _Args(_Call):
    """A kept call of an entry point that takes no workspace; ``pair``: the two tensors that it writes."""

    __slots__ = ("pair", "gap", "apart")

    def __init__(self, key, args, pair=None):
        args.struct_size = ctypes.sizeof(args)
        super().__init__(key, 0, args)
        self.pair = pair and (_reach(pair[0]), _reach(pair[1]))
        # distances of addresses at which they were last seen to be apart (shapes and strides are in the key): of the pair,
        # and of what is read beside an output
        self.gap = self.apart = None

    def check_pair(self, first, second, gap, names):
        """Refuses written tensors, at this distance, that share an element."""
        if gap < self.pair[0] and -gap < self.pair[1] and not _apart(first, second):
            raise ValueError(f"{names} must be different tensors, and share no element")
        self.gap = gap

    def launch(self, entry, device, stream):
        _launch(device, entry, *self.refs, stream)


# (0.1 us a call instead of 0.4 through _lib.current_stream_handle, which asks what a GPU tensor's device answers)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _stream(t):
    """The current stream of a tensor's device; None where it is no GPU tensor (the checks say so)."""
    return _raw_stream(t.device.index) if isinstance(t, torch.Tensor) and t.is_cuda else None


def _meta(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def fused_rope_kv_append_fp4(q, k, v, k_cache, v_cache, block_ids, block_offsets, positions, rotary_dim=None,
                             base=10_000.0, cos_sin_table=None, q_out=None, check_indices=True):
    """Rotate Q/K and append K/V to a 4-bit cache through one HIP kernel; returns the rotated Q.

    ``q`` ``[tokens, num_q_heads, head_dim]``, ``k`` and ``v`` ``[tokens,
    num_kv_heads, head_dim]``, float16 or bfloat16, any strides but a unit dim
    stride (slices of one projection are taken as they are).  Token ``t`` goes to
    block ``block_ids[t]``, place ``block_offsets[t]``; a slot may occur once.
    ``rotary_dim``, ``base`` and ``cos_sin_table`` as in
    :func:`flashdec_amd.fused_rope_kv_append`, whose rotation this is; K is
    quantised from the 32-bit result, V from its 16-bit values.  ``q_out`` may share a
    buffer with ``q``, ``k`` and ``v``, and no element of them.

    ``check_indices=True`` checks the index values first, which waits for the
    stream.  ``False`` (a step with the cache's own indices, a captured call) checks
    nothing: tokens whose slot is outside the cache are then not stored, and
    positions outside a table read its nearest row.
    """
    rotary_dim = q.shape[-1] if rotary_dim is None and isinstance(q, torch.Tensor) and q.dim() else rotary_dim
    base, key = float(base), None
    try:  # (one flat tuple: with a tuple a tensor a call takes 1.5 us more)
        key = (type(rotary_dim), rotary_dim, base, q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype,
               k.device, v.shape, v.stride(), v.dtype, v.device, k_cache.shape, k_cache.stride(), k_cache.dtype,
               k_cache.device, v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.device, block_ids.shape,
               block_ids.stride(), block_ids.dtype, block_ids.device, block_offsets.shape, block_offsets.stride(),
               block_offsets.dtype, block_offsets.device, positions.shape, positions.stride(), positions.dtype,
               positions.device, _meta(cos_sin_table), _meta(q_out))
    except AttributeError:  # an argument that is no tensor: the checks say which
        pass
    call = _kept("fp4_append", key)
    if call is None:
        if not isinstance(q, torch.Tensor):  # (without one the checks are those of an append without rotation)
            raise TypeError("q must be a torch.Tensor")
        args = _append_args(q, k, v, k_cache, v_cache, block_ids, block_offsets, positions, rotary_dim, base, cos_sin_table,
                            q_out)
        call = _keep("fp4_append", _Args(key, args, (k_cache, v_cache)))
        call.reach = None if q_out is None else (_reach(q_out), _reach(q), _reach(k), _reach(v))
    args = call.args
    if q_out is None:
        q_out = q.new_empty(q.shape)
    if args.num_tokens == 0:
        return q_out
    old, new = q.data_ptr(), q_out.data_ptr()
    if call.reach is not None:  # (of a q_out that is the caller's)
        gaps = new - old, new - k.data_ptr(), new - v.data_ptr()
        if gaps != call.apart:
            end, *reaches = call.reach
            for t, reach, gap in zip((q, k, v), reaches, gaps):
                if gap < reach and -gap < end and not _apart(t, q_out):
                    raise ValueError("q_out must lie apart from q, k and v")
            call.apart = gaps
    if check_indices:
        rows = -1 if cos_sin_table is None else cos_sin_table.shape[1]
        if _validate_index_values(block_ids, block_offsets, positions, k_cache.shape[0], args.block_size, rows):
            raise ValueError("positions must be below the cos_sin_table's rows")
    args.q, args.q_out, args.positions = old, new, positions.data_ptr()
    if cos_sin_table is not None:
        args.cos_sin_table = cos_sin_table.data_ptr()
    _append(call, k, v, k_cache, v_cache, block_ids, block_offsets)
    return q_out


def kv_append_fp4(k, v, k_cache, v_cache, block_ids, block_offsets, check_indices=True):
    """:func:`fused_rope_kv_append_fp4` of keys that need no rotation: K and V quantised into their slots."""
    key = None
    try:
        key = (k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device, k_cache.shape,
               k_cache.stride(), k_cache.dtype, k_cache.device, v_cache.shape, v_cache.stride(), v_cache.dtype,
               v_cache.device, block_ids.shape, block_ids.stride(), block_ids.dtype, block_ids.device, block_offsets.shape,
               block_offsets.stride(), block_offsets.dtype, block_offsets.device)
    except AttributeError:
        pass
    call = _kept("fp4_kv_append", key)
    if call is None:
        call = _keep("fp4_kv_append", _Args(key, _append_args(None, k, v, k_cache, v_cache, block_ids, block_offsets, None,
                                                              0, 1.0, None, None), (k_cache, v_cache)))
    if call.args.num_tokens == 0:
        return
    if check_indices:
        _validate_index_values(block_ids, block_offsets, None, k_cache.shape[0], call.args.block_size)
    _append(call, k, v, k_cache, v_cache, block_ids, block_offsets)


def _append(call, k, v, k_cache, v_cache, block_ids, block_offsets):
    args, device = call.args, k_cache.device
    args.k, args.v = k.data_ptr(), v.data_ptr()
    gap = _point_pools(args, k_cache, v_cache)
    if gap != call.gap:
        call.check_pair(k_cache, v_cache, gap, "k_cache and v_cache")
    args.block_ids, args.block_offsets = block_ids.data_ptr(), block_offsets.data_ptr()
    call.launch(_lib.fp4_append, device, _raw_stream(device.index))


def _point_pools(args, k_cache, v_cache):
    """The pools' addresses, with what a kept call's key does not hold: that they lie on 16-byte lines.  Returns their
    distance."""
    k, v = k_cache.data_ptr(), v_cache.data_ptr()
    if (k | v) % 16:
        raise ValueError("the caches' blocks must be contiguous and lie on 16-byte lines")
    args.k_cache, args.v_cache = k, v
    return v - k


def _append_args(q, k, v, k_cache, v_cache, block_ids, block_offsets, positions, rotary_dim, base, table, q_out):
    if not isinstance(k, torch.Tensor):
        raise TypeError("k must be a torch.Tensor")
    if k.dim() != 3:
        raise ValueError("q, k, and v must have shape [tokens, heads, head_dim]")
    if not k.is_cuda:
        raise ValueError("k must be a CUDA tensor")
    if k.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("a 4-bit cache is appended to from float16 and bfloat16 tensors")
    device, (tokens, num_kv_heads, head_dim) = k.device, k.shape
    block_size = _check_pools(k_cache, v_cache, head_dim, device)
    _check_written((k_cache, v_cache))
    if k_cache.shape[1] != num_kv_heads:
        raise ValueError("k and v must have the cache's num_kv_heads")
    for name, t, heads in (("k", k, num_kv_heads), ("v", v, num_kv_heads)):
        _check_rows(name, t, tokens, heads, head_dim, k.dtype, device)
    _check_indices(tokens, device, block_ids=block_ids, block_offsets=block_offsets)
    args = _lib.Fp4AppendArgs()
    if q is not None or rotary_dim:
        _check_rows("q", q, tokens, None, head_dim, k.dtype, device)
        if q_out is not None:
            _check_rows("q_out", q_out, tokens, q.shape[1], head_dim, k.dtype, device)
            if not _spread_out(q_out):
                raise ValueError("q_out must have no overlapping elements")
        if q.shape[1] < 1:
            raise ValueError("num_q_heads must be positive")
        _check_indices(tokens, device, positions=positions)
        if isinstance(rotary_dim, bool) or not isinstance(rotary_dim, int):
            raise ValueError("rotary_dim must be an even integer")
        if rotary_dim <= 0 or rotary_dim > head_dim or rotary_dim % 2 != 0:
            raise ValueError("rotary_dim must be positive, even, and no larger than head_dim")
        if not math.isfinite(base) or base <= 0.0:
            raise ValueError("base must be a positive finite number")
        if table is not None:
            _check_cos_sin_table(table, rotary_dim, device)
            args.table_rows = table.shape[1]
        args.num_q_heads, args.rotary_dim, args.base = q.shape[1], rotary_dim, base
        args.q_stride[:] = q.stride()[:2]
        args.q_out_stride[:] = (q.shape[1] * head_dim, head_dim) if q_out is None else q_out.stride()[:2]
        args.index_dtype[2] = _lib.index_code(positions.dtype)
    args.dtype = _lib.dtype_code(k.dtype)
    args.num_tokens, args.num_kv_heads, args.head_dim = tokens, num_kv_heads, head_dim
    args.block_size, args.num_blocks = block_size, k_cache.shape[0]
    args.k_stride[:], args.v_stride[:] = k.stride()[:2], v.stride()[:2]
    args.k_cache_stride[:], args.v_cache_stride[:] = k_cache.stride()[:2], v_cache.stride()[:2]
    args.index_dtype[0], args.index_dtype[1] = _lib.index_code(block_ids.dtype), _lib.index_code(block_offsets.dtype)
    return args


def paged_kv_read_fp4(k_cache, v_cache, block_ids, block_offsets, head_dim, dtype=torch.bfloat16):
    """The tokens at ``(block_ids[t], block_offsets[t])`` of a 4-bit cache as 16-bit ``(k, v)``, each ``[tokens,
    num_kv_heads, head_dim]``: exact in bfloat16.  Slots outside the cache give zeros."""
    if not isinstance(k_cache, torch.Tensor) or not isinstance(block_ids, torch.Tensor):
        raise TypeError("k_cache and block_ids must be torch.Tensors")
    if k_cache.dim() != 3 or block_ids.dim() != 1:
        raise ValueError("k_cache must be a 3D and block_ids a 1D tensor")
    shape = (block_ids.shape[0], k_cache.shape[1], head_dim)
    k, v = k_cache.new_empty(shape, dtype=dtype), k_cache.new_empty(shape, dtype=dtype)
    return paged_kv_read_fp4_into(k_cache, v_cache, block_ids, block_offsets, k, v)


def paged_kv_read_fp4_into(k_cache, v_cache, block_ids, block_offsets, k_out, v_out):
    """:func:`paged_kv_read_fp4` into ``k_out`` and ``v_out`` (unit dim stride); returns them."""
    key = None
    try:
        key = (k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.device, v_cache.shape, v_cache.stride(), v_cache.dtype,
               v_cache.device, block_ids.shape, block_ids.stride(), block_ids.dtype, block_ids.device, block_offsets.shape,
               block_offsets.stride(), block_offsets.dtype, block_offsets.device, k_out.shape, k_out.stride(), k_out.dtype,
               k_out.device, v_out.shape, v_out.stride(), v_out.dtype, v_out.device)
    except AttributeError:
        pass
    call = _kept("fp4_read", key)
    if call is None:
        call = _keep("fp4_read", _Args(key, _read_args(k_cache, v_cache, block_ids, block_offsets, k_out, v_out),
                                       (k_out, v_out)))
    args, device = call.args, k_cache.device
    if args.num_tokens == 0:
        return k_out, v_out
    _point_pools(args, k_cache, v_cache)
    args.block_ids, args.block_offsets = block_ids.data_ptr(), block_offsets.data_ptr()
    first, second = k_out.data_ptr(), v_out.data_ptr()
    args.k_out, args.v_out = first, second
    if second - first != call.gap:
        call.check_pair(k_out, v_out, second - first, "k_out and v_out")
    call.launch(_lib.fp4_read, device, _raw_stream(device.index))
    return k_out, v_out


def _read_args(k_cache, v_cache, block_ids, block_offsets, k_out, v_out):
    if not isinstance(k_out, torch.Tensor):
        raise TypeError("k_out must be a torch.Tensor")
    if k_out.dim() != 3:
        raise ValueError("k_out and v_out must have shape [tokens, num_kv_heads, head_dim]")
    if not k_out.is_cuda:
        raise ValueError("k_out must be a CUDA tensor")
    if k_out.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("a 4-bit cache is read as float16 or bfloat16")
    device, (tokens, num_kv_heads, head_dim) = k_out.device, k_out.shape
    block_size = _check_pools(k_cache, v_cache, head_dim, device)
    if k_cache.shape[1] != num_kv_heads:
        raise ValueError("k_out and v_out must have the cache's num_kv_heads")
    _check_indices(tokens, device, block_ids=block_ids, block_offsets=block_offsets)
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        _check_rows(name, t, tokens, num_kv_heads, head_dim, k_out.dtype, device)
        if not _spread_out(t):
            raise ValueError(f"{name} must have no overlapping elements")
    args = _lib.Fp4ReadArgs()
    args.dtype = _lib.dtype_code(k_out.dtype)
    args.num_tokens, args.num_kv_heads, args.head_dim = tokens, num_kv_heads, head_dim
    args.block_size, args.num_blocks = block_size, k_cache.shape[0]
    args.k_cache_stride[:], args.v_cache_stride[:] = k_cache.stride()[:2], v_cache.stride()[:2]
    args.index_dtype[:] = _lib.index_code(block_ids.dtype), _lib.index_code(block_offsets.dtype)
    args.k_out_stride[:], args.v_out_stride[:] = k_out.stride()[:2], v_out.stride()[:2]
    return args


def paged_decode_attention_fp4(q, k_cache, v_cache, block_tables, seq_lens, sm_scale=None, kv_reuse=False, ragged=False):
    """Single-token decode attention over a 4-bit cache: :func:`flashdec_amd.paged_decode_attention` of the values that
    it holds.

    ``q`` ``[num_seqs, num_q_heads, head_dim]`` (float16 or bfloat16, any
    strides), ``block_tables`` ``[num_seqs, max_blocks_per_seq]`` and ``seq_lens``
    ``[num_seqs]`` (int32 or int64).  Tokens in blocks outside the pool are not
    attended; a row with nothing to attend gives zeros.  ``ragged=True`` says that the
    rows' lengths vary widely (one may be many times another): long rows are then cut
    finer in batches of up to 256 that would otherwise give each its own workgroups.  Returns
    ``[num_seqs, num_q_heads, head_dim]`` in q.dtype.
    """
    if not isinstance(q, torch.Tensor):
        raise TypeError("q must be a torch.Tensor")
    return paged_decode_attention_fp4_into(q, k_cache, v_cache, block_tables, seq_lens, torch.empty_like(q), sm_scale,
                                           kv_reuse, ragged)


def paged_decode_attention_fp4_into(q, k_cache, v_cache, block_tables, seq_lens, out, sm_scale=None, kv_reuse=False,
                                    ragged=False):
    """:func:`paged_decode_attention_fp4` into ``out`` (any strides); returns it.

    ``kv_reuse=True``: rows share blocks (a common prefix), so the cache is read
    with plain, cached loads; the result is the same.  ``sm_scale`` is read at
    every call (of an array or a tensor, the value that it then holds).
    """
    sm_scale, kv_reuse, ragged = _number(sm_scale, float), bool(kv_reuse), bool(ragged)
    stream, key = _stream(q), None
    try:
        key = (stream, sm_scale, kv_reuse, ragged, q.shape, q.stride(), q.dtype, q.device, k_cache.shape,
               k_cache.stride(), k_cache.dtype, k_cache.device, v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.device,
               block_tables.shape, block_tables.stride(), block_tables.dtype, block_tables.device, seq_lens.shape,
               seq_lens.stride(), seq_lens.dtype, seq_lens.device, out.shape, out.stride(), out.dtype, out.device)
    except AttributeError:
        pass
    call = _kept("fp4_decode", key)
    if call is None:
        args = _decode_args(q, k_cache, v_cache, block_tables, seq_lens, out, sm_scale, kv_reuse, ragged)
        call = _keep("fp4_decode", _Call(key, _launch(q.device, _lib.fp4_decode_floats, args), args))
    else:
        args = call.args
        args.q, args.out = q.data_ptr(), out.data_ptr()
        _point_pools(args, k_cache, v_cache)
        args.block_tables, args.seq_lens = block_tables.data_ptr(), seq_lens.data_ptr()
    call.launch(_lib.fp4_decode, q.device, stream)
    return out


def _check_heads(q, pool):
    if q.shape[0] <= 0 or q.shape[1] <= 0:
        raise ValueError("num_seqs and num_q_heads must be positive")
    if q.shape[1] % pool.shape[1] != 0:
        raise ValueError("num_q_heads must be divisible by num_kv_heads")


def _check_tables(block_tables, seq_lens, num_seqs):
    if block_tables.dim() != 2 or seq_lens.dim() != 1 or block_tables.shape[0] != num_seqs or seq_lens.numel() != num_seqs:
        raise ValueError("block_tables and seq_lens must have one row/value per sequence")
    if block_tables.shape[1] <= 0:
        raise ValueError("max_blocks_per_seq must be positive")
    for name, t in (("block_tables", block_tables), ("seq_lens", seq_lens)):
        if t.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name} must be int32 or int64")


def _decode_args(q, k_cache, v_cache, block_tables, seq_lens, out, sm_scale, kv_reuse, ragged):
    for name, t in (("q", q), ("block_tables", block_tables), ("seq_lens", seq_lens), ("out", out)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")
        if t.device != q.device:
            raise ValueError("the caches and the other tensors must be on the same CUDA device")
    if q.dim() != 3:
        raise ValueError("q must have shape [num_seqs, num_q_heads, head_dim]")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("paged_decode_attention_fp4 supports float16 and bfloat16 queries")
    num_seqs, num_q_heads, head_dim = q.shape
    block_size = _check_pools(k_cache, v_cache, head_dim, q.device)
    _check_heads(q, k_cache)
    _check_out(out, q)
    _check_tables(block_tables, seq_lens, num_seqs)
    args = _lib.Fp4DecodeArgs()
    args.dtype = _lib.dtype_code(q.dtype)
    args.num_seqs, args.num_q_heads, args.num_kv_heads = num_seqs, num_q_heads, k_cache.shape[1]
    args.head_dim, args.block_size, args.num_blocks = head_dim, block_size, k_cache.shape[0]
    args.max_blocks_per_seq = block_tables.shape[1]
    args.q, args.out = q.data_ptr(), out.data_ptr()
    args.q_stride[:], args.out_stride[:] = q.stride(), out.stride()
    args.k_cache, args.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    args.k_cache_stride[:], args.v_cache_stride[:] = k_cache.stride()[:2], v_cache.stride()[:2]
    args.block_tables, args.seq_lens = block_tables.data_ptr(), seq_lens.data_ptr()
    args.block_tables_dtype, args.seq_lens_dtype = _lib.index_code(block_tables.dtype), _lib.index_code(seq_lens.dtype)
    args.block_tables_stride[:], args.seq_lens_stride = block_tables.stride(), seq_lens.stride(0)
    args.sm_scale = 1.0 / math.sqrt(head_dim) if sm_scale is None else sm_scale
    args.kv_reuse, args.ragged = 1 if kv_reuse else 0, 1 if ragged else 0
    return args
