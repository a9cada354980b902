"""Attention over the blocks that matter, on MI355X through ``libflashdec_hip.so``.

Most of a long context's tokens weigh nothing in a decode step.  Each KV head can
attend a fixed number of its row's blocks instead, those that may hold the largest
products with the step's queries (no counterpart in the reference, whose decode
attends every cached token):

* :func:`paged_key_bounds` keeps, for every complete block, the least and the largest
  key in each dim;
* :func:`paged_block_select` scores the blocks by them, an upper bound of what their
  keys give, and takes the best for each row and KV head, with the row's first and
  last blocks;
* :func:`paged_decode_attention_blocks` attends the tokens of the chosen blocks.

A step, for a context of any length::

    bounds = torch.empty((num_blocks, num_kv_heads, 2, head_dim), device="cuda", dtype=k_cache.dtype)
    ...
    fused_rope_kv_append(q, k, v, k_cache, v_cache, block_ids, block_offsets, positions)
    paged_key_bounds(k_cache, block_tables, seq_lens, bounds, new_tokens=1)  # lengths with the new token
    chosen = paged_block_select(q_rot, k_cache, bounds, block_tables, seq_lens, 128, sink_blocks=1, recent_blocks=4)
    out = paged_decode_attention_blocks(q_rot, k_cache, v_cache, chosen)

All three take a cache held in 4 bits (:mod:`flashdec_amd.fp4`) as well.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .bounded import _Call, _block_size, _keep, _kept, _launch, _number, _spread_out, _whole
from . import fp4
from .fp4 import _Args, _raw_stream, _stream
from .paged_decode import (
    _cache_strides,
    _capturing,
    _decode_args,
    _even_workspace,
    _layout_axes,
    _held_workspace,
    _off_16,
    _split_workspace,
    _validate_inputs,
)


class BlockSelection(NamedTuple):
    """What :func:`paged_block_select` chose, for each row and KV head, int32.

    ``blocks`` ``[num_seqs, num_kv_heads, n]``: indices of the row's chosen blocks,
    ascending, -1 behind the last.  ``tables`` (the same shape): their ids as blocks
    of one KV head, ``id * block_step + head``.  ``lens`` ``[num_seqs,
    num_kv_heads]``: tokens in them.  ``block_step``: KV-head blocks from one block
    of the pool to the next.
    """

    blocks: torch.Tensor
    tables: torch.Tensor
    lens: torch.Tensor
    block_step: int


def _block_step(cache):
    """KV-head blocks from one block of a pool to the next: the pool seen as blocks of one KV head each."""
    if cache.shape[1] == 1:
        return 1
    step, rest = divmod(cache.stride(0), cache.stride(1)) if cache.stride(1) > 0 else (0, 1)
    if rest or step < cache.shape[1]:
        raise ValueError("the cache's block stride must be a multiple of its KV head stride that holds every head")
    return step


def _is_fp4(cache):
    return isinstance(cache, torch.Tensor) and cache.dtype == torch.uint8


def _check_bounds(bounds, k_cache, head_dim, dtype):
    if bounds.dim() != 4 or tuple(bounds.shape) != (k_cache.shape[0], k_cache.shape[1], 2, head_dim):
        raise ValueError("bounds must have shape [num_blocks, num_kv_heads, 2, head_dim]")
    if bounds.dtype != dtype:
        raise ValueError("bounds must have the cache's dtype, and that of the queries")
    if bounds.device != k_cache.device:
        raise ValueError("bounds must be on the cache's device")
    if not bounds.is_contiguous():
        raise ValueError("bounds must be contiguous")


def _on_line(bounds):
    """The bounds' address, which a kept call's key does not hold."""
    at = bounds.data_ptr()
    if at % 16:
        raise ValueError("bounds must lie on a 16-byte line")
    return at


def _tensors(**tensors):
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")


def _check_row_tensors(k_cache, block_tables, seq_lens, block_size, kv_layout, q=None):
    """The decode call's checks, on a query of one head per KV head where there is none; returns (block size, dim axis)."""
    token_axis, dim_axis = _layout_axes(kv_layout)
    block_size = _block_size(k_cache, block_size, token_axis)
    if k_cache.dim() != 4:
        raise ValueError("k_cache must be a 4D tensor")
    if q is None:
        rows = block_tables.shape[0] if block_tables.dim() == 2 else 1
        q = k_cache.new_empty((rows, k_cache.shape[1], k_cache.shape[dim_axis]))
    _validate_inputs(q, k_cache, k_cache, block_tables, seq_lens, block_size, 2, None, kv_layout)
    return block_size, dim_axis


def _fill_rows(args, block_tables, seq_lens):
    args.num_seqs, args.max_blocks_per_seq = block_tables.shape
    args.block_tables_dtype, args.seq_lens_dtype = _lib.index_code(block_tables.dtype), _lib.index_code(seq_lens.dtype)
    args.block_tables_stride[:], args.seq_lens_stride = block_tables.stride(), seq_lens.stride(0)


def paged_key_bounds(k_cache, block_tables, seq_lens, bounds, new_tokens=None, block_size=None, kv_layout="token_major"):
    """Brings ``bounds`` up to date with the rows' last ``new_tokens`` tokens (None: all); returns it.

    ``bounds`` ``[num_blocks, num_kv_heads, 2, head_dim]`` in the cache's dtype (of a
    4-bit cache: the queries'), contiguous: plane 0 the least, plane 1 the largest key of a block in each dim
    (NaN where a key is).  Blocks that are complete and hold one of those tokens are
    written; others stay as they are, the partly filled last one too, which is never
    scored.  A row that fewer tokens were added to than ``new_tokens`` has some blocks
    written again, to the same values.  Tokens that move within their blocks
    (:func:`flashdec_amd.paged_kv_evict`) leave the bounds as they were: call again for
    the whole row.  Cache and tables as in :func:`flashdec_amd.paged_decode_attention`.
    """
    block_size = _number(block_size, int)
    key = None
    try:
        key = (type(new_tokens), new_tokens, block_size, kv_layout, k_cache.shape, k_cache.stride(), k_cache.dtype,
               k_cache.device, block_tables.shape, block_tables.stride(), block_tables.dtype, block_tables.device,
               seq_lens.shape, seq_lens.stride(), seq_lens.dtype, seq_lens.device, bounds.shape, bounds.stride(),
               bounds.dtype, bounds.device)
    except AttributeError:  # an argument that is no tensor: the checks say which
        pass
    call = _kept("key_bounds", key)
    if call is None:
        _tensors(k_cache=k_cache, block_tables=block_tables, seq_lens=seq_lens, bounds=bounds)
        call = _keep("key_bounds", _Args(key, _bounds_args(k_cache, block_tables, seq_lens, bounds, new_tokens, block_size,
                                                           kv_layout)))
    args, device = call.args, k_cache.device
    args.k_cache, args.bounds = k_cache.data_ptr(), _on_line(bounds)
    args.block_tables, args.seq_lens = block_tables.data_ptr(), seq_lens.data_ptr()
    call.launch(_lib.key_bounds, device, _raw_stream(device.index))
    return bounds


def _bounds_args(k_cache, block_tables, seq_lens, bounds, new_tokens, block_size, kv_layout):
    args = _lib.KeyBoundsArgs()
    if _is_fp4(k_cache):
        if bounds.dim() != 4 or bounds.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("bounds of a 4-bit cache must be float16 or bfloat16, [num_blocks, num_kv_heads, 2, head_dim]")
        head_dim, rows = bounds.shape[3], block_tables.shape[0] if block_tables.dim() == 2 else 1
        block_size = _check_fp4_rows(k_cache, block_tables, seq_lens, rows, head_dim, block_size, kv_layout)
        _check_bounds(bounds, k_cache, head_dim, bounds.dtype)
        args.fp4 = 1
        args.k_stride[:2] = k_cache.stride()[:2]
    else:
        block_size, dim_axis = _check_row_tensors(k_cache, block_tables, seq_lens, block_size, kv_layout)
        head_dim = k_cache.shape[dim_axis]
        _check_bounds(bounds, k_cache, head_dim, k_cache.dtype)
        args.k_stride[:] = _cache_strides(k_cache, 5 - dim_axis, dim_axis)
    args.dtype = _lib.dtype_code(bounds.dtype)
    args.num_kv_heads, args.head_dim, args.block_size = k_cache.shape[1], head_dim, block_size
    args.num_blocks = k_cache.shape[0]
    _fill_rows(args, block_tables, seq_lens)
    args.new_tokens = 2**62 if new_tokens is None else min(_whole(new_tokens, "new_tokens", 0), 2**62)
    return args


def _check_fp4_rows(pool, block_tables, seq_lens, num_seqs, head_dim, block_size, kv_layout):
    """The 4-bit decode call's checks of a pool and its rows; returns the block size."""
    if not pool.is_cuda:
        raise ValueError("the cache must be a CUDA tensor")
    found = fp4._check_pools(pool, pool, head_dim, pool.device)
    if kv_layout != "token_major":
        raise ValueError("a 4-bit cache has kv_layout 'token_major'")
    if block_size is not None and block_size != found:
        raise ValueError("block_size must match the cache's shape")
    if any(t.device != pool.device for t in (block_tables, seq_lens)):
        raise ValueError("the cache, block_tables and seq_lens must be on the same CUDA device")
    fp4._check_tables(block_tables, seq_lens, num_seqs)
    if num_seqs <= 0:
        raise ValueError("num_seqs must be positive")
    return found


def paged_block_select(q, k_cache, bounds, block_tables, seq_lens, num_select, sink_blocks=1, recent_blocks=1,
                       block_size=None, kv_layout="token_major"):
    """The ``num_select`` blocks of each row and KV head that ``q`` attends, as a :class:`BlockSelection`.

    A row of ``num_select`` blocks or fewer keeps all.  Of a longer one each KV head
    keeps the first ``sink_blocks``, the last ``recent_blocks`` (at least one) and, of
    those between, the ones with the highest score: the sum over its query heads and
    over the dims of ``max(q lo, q hi)``, ``lo`` and ``hi`` the block's ``bounds``,
    summed in 64 bits and rounded to 32 (equal scores: the lower index; NaN first, as
    where an infinite bound meets queries that are all on the other side of zero).
    With no place left between them (``num_select == sink_blocks + recent_blocks``)
    nothing is scored, and ``bounds`` are not read.
    ``sm_scale`` does not enter: it is taken to be positive.  ``k_cache`` says how the
    pool is laid out and is not read; the values' pool must be laid out like it.
    """
    _tensors(k_cache=k_cache, block_tables=block_tables)
    if block_tables.dim() != 2 or k_cache.dim() != (3 if _is_fp4(k_cache) else 4):
        raise ValueError("block_tables must be a 2D tensor, and k_cache a 4D one (of a 4-bit cache 3D)")
    shape = (block_tables.shape[0], k_cache.shape[1], _whole(num_select, "num_select", 1))
    blocks, tables = (torch.empty(shape, device=k_cache.device, dtype=torch.int32) for _ in range(2))
    lens = torch.empty(shape[:2], device=k_cache.device, dtype=torch.int32)
    return paged_block_select_into(q, k_cache, bounds, block_tables, seq_lens, blocks, tables, lens, sink_blocks,
                                   recent_blocks, block_size, kv_layout)


def paged_block_select_into(q, k_cache, bounds, block_tables, seq_lens, blocks, tables, lens, sink_blocks=1,
                            recent_blocks=1, block_size=None, kv_layout="token_major"):
    """:func:`paged_block_select` into contiguous int32 ``blocks``, ``tables`` ``[num_seqs, num_kv_heads, num_select]`` and
    ``lens`` ``[num_seqs, num_kv_heads]``."""
    block_size = _number(block_size, int)
    stream, key = _stream(q), None
    try:
        key = (stream, type(sink_blocks), type(recent_blocks), sink_blocks, recent_blocks, block_size, kv_layout, q.shape,
               q.stride(), q.dtype, q.device, k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.device, bounds.shape,
               bounds.stride(), bounds.dtype, bounds.device, block_tables.shape, block_tables.stride(), block_tables.dtype,
               block_tables.device, seq_lens.shape, seq_lens.stride(), seq_lens.dtype, seq_lens.device, blocks.shape,
               blocks.stride(), blocks.dtype, blocks.device, tables.shape, tables.stride(), tables.dtype, tables.device,
               lens.shape, lens.stride(), lens.dtype, lens.device)
    except AttributeError:
        pass
    call = _kept("block_select", key)
    if call is None:
        _tensors(q=q, k_cache=k_cache, bounds=bounds, block_tables=block_tables, seq_lens=seq_lens, blocks=blocks,
                 tables=tables, lens=lens)
        args = _select_args(q, k_cache, bounds, block_tables, seq_lens, blocks, tables, lens, sink_blocks, recent_blocks,
                            block_size, kv_layout)
    else:
        args = call.args
    args.q, args.bounds = q.data_ptr(), _on_line(bounds)
    args.block_tables, args.seq_lens = block_tables.data_ptr(), seq_lens.data_ptr()
    first, second, third = blocks.data_ptr(), tables.data_ptr(), lens.data_ptr()
    args.blocks, args.tables, args.lens = first, second, third
    gaps = second - first, third - first
    if call is None or call.reach != gaps:  # (the last call's distances are looked at once)
        size, count = 4 * blocks.numel(), 4 * lens.numel()  # (all are contiguous)
        if abs(first - second) < size or -count < third - first < size or -count < third - second < size:
            raise ValueError("blocks, tables and lens must be different tensors, and share no element")
        if call is None:
            call = _keep("block_select", _Call(key, _launch(q.device, _lib.block_select_words, args), args))
        call.reach = gaps
    call.launch(_lib.block_select, q.device, stream)
    return BlockSelection(blocks, tables, lens, args.block_step)


def _select_args(q, k_cache, bounds, block_tables, seq_lens, blocks, tables, lens, sink_blocks, recent_blocks, block_size,
                 kv_layout):
    if _is_fp4(k_cache):
        if q.dim() != 3 or q.dtype not in (torch.float16, torch.bfloat16) or q.device != k_cache.device:
            raise ValueError("q must be float16 or bfloat16, [num_seqs, num_q_heads, head_dim], on the cache's device")
        block_size = _check_fp4_rows(k_cache, block_tables, seq_lens, q.shape[0], q.shape[2], block_size, kv_layout)
        fp4._check_heads(q, k_cache)
    else:
        block_size, _ = _check_row_tensors(k_cache, block_tables, seq_lens, block_size, kv_layout, q)
    num_seqs, num_q_heads, head_dim = q.shape
    num_kv_heads = k_cache.shape[1]
    _check_bounds(bounds, k_cache, head_dim, q.dtype)
    _whole(sink_blocks, "sink_blocks", 0)
    _whole(recent_blocks, "recent_blocks", 1)
    outs = (blocks, tables, lens)
    if blocks.dim() != 3 or blocks.shape[:2] != (num_seqs, num_kv_heads) or blocks.shape[2] < 1:
        raise ValueError("blocks must have shape [num_seqs, num_kv_heads, num_select]")
    if tables.shape != blocks.shape or lens.shape != blocks.shape[:2]:
        raise ValueError("tables must have the shape of blocks, and lens its first two dims")
    if any(t.dtype != torch.int32 or not t.is_contiguous() or t.device != q.device for t in outs):
        raise ValueError("blocks, tables and lens must be contiguous int32 tensors on the cache's device")
    if sink_blocks + recent_blocks > blocks.shape[2]:
        raise ValueError("num_select must hold sink_blocks and recent_blocks")
    args = _lib.BlockSelectArgs()
    args.dtype = _lib.dtype_code(q.dtype)
    args.num_q_heads, args.num_kv_heads, args.head_dim = num_q_heads, num_kv_heads, head_dim
    args.block_size, args.num_blocks = block_size, k_cache.shape[0]
    args.q_stride[:] = q.stride()
    _fill_rows(args, block_tables, seq_lens)
    args.select, args.sink_blocks, args.recent_blocks = blocks.shape[2], sink_blocks, recent_blocks
    args.block_step = _block_step(k_cache)
    return args


def paged_decode_attention_blocks(q, k_cache, v_cache, selection, sm_scale=None, block_size=None, kv_layout="token_major",
                                  kv_reuse=False, ragged=False):
    """Decode attention over the blocks of a :class:`BlockSelection`, of each KV head its own.

    ``q`` and the caches as in :func:`flashdec_amd.paged_decode_attention`; both
    caches laid out as the one that the selection was made for.  A row with nothing
    chosen gives zeros.  ``ragged=True`` says that the rows' numbers of chosen tokens
    vary widely (a batch with rows far below ``num_select`` blocks).
    Returns ``[num_seqs, num_q_heads, head_dim]`` in q.dtype.
    """
    _tensors(q=q)
    return paged_decode_attention_blocks_into(q, k_cache, v_cache, selection, torch.empty_like(q), sm_scale, block_size,
                                              kv_layout, kv_reuse, ragged)


def paged_decode_attention_blocks_into(q, k_cache, v_cache, selection, out, sm_scale=None, block_size=None,
                                       kv_layout="token_major", kv_reuse=False, ragged=False):
    """:func:`paged_decode_attention_blocks` into ``out``; returns it."""
    if not isinstance(selection, BlockSelection):
        raise TypeError("selection must be a BlockSelection")
    tables, lens = selection.tables, selection.lens
    sm_scale, block_size, ragged, kv_reuse = _number(sm_scale, float), _number(block_size, int), bool(ragged), bool(kv_reuse)
    stream, key = _stream(q), None
    try:
        # (whether a pointer is off the 16-byte lines, too: the plan depends on it)
        key = (stream, sm_scale, block_size, kv_layout, ragged, kv_reuse, selection.block_step, q.shape, q.stride(), q.dtype,
               q.device, k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.device, v_cache.shape, v_cache.stride(),
               v_cache.dtype, v_cache.device, tables.shape, tables.stride(), tables.dtype, tables.device, lens.shape,
               lens.stride(), lens.dtype, lens.device, out.shape, out.stride(), out.dtype, out.device,
               _off_16(q, k_cache, v_cache, None, None))
    except (AttributeError, TypeError):
        pass
    if _is_fp4(k_cache):
        return _fp4_blocks(q, k_cache, v_cache, selection, out, sm_scale, block_size, kv_layout, kv_reuse, ragged)
    call = None if _capturing(stream or 0) else _kept("blocks", key)  # (a captured call's partials are the graph's own)
    if call is None:
        _check_blocks(q, k_cache, v_cache, selection, out)
        # each KV head of a row as a request of its own, over the pool seen as blocks of one KV head
        rows, group, head_dim = tables.shape[0] * tables.shape[1], q.shape[1] // k_cache.shape[1], q.shape[2]
        heads = [_one_head_blocks(cache, selection.block_step) for cache in (k_cache, v_cache)]
        flat = _rows_flat(q) and _rows_flat(out)
        queries = q.reshape(rows, group, head_dim)
        result = out.view(queries.shape) if _rows_flat(out) else torch.empty_like(queries)
        args, _ = _decode_args(queries, *heads, tables.view(rows, -1), lens.view(rows), result, sm_scale, block_size, 2,
                               kv_layout, None, None, 1, None, None, None, ragged, kv_reuse, even=True)
        if flat and not args.captured_workspace:
            _keep("blocks", _Blocks(key, args))
    else:
        args = call.args
        if args.library_workspace:
            call.point_workspace(q.device, stream)
        args.q, args.k_cache, args.v_cache = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
        args.block_tables, args.seq_lens, args.out = tables.data_ptr(), lens.data_ptr(), out.data_ptr()
    if args.even:
        workspace = _even_workspace(q.device, args.even, stream)
        _launch(q.device, _lib.paged_decode_even, args, workspace.data_ptr(), args.even, stream)
    else:
        _launch(q.device, _lib.paged_decode, args, stream)
    if call is None and not _rows_flat(out):
        out.copy_(result.view(out.shape))
    return out


def _fp4_blocks(q, k_cache, v_cache, selection, out, sm_scale, block_size, kv_layout, kv_reuse, ragged):
    _check_blocks(q, k_cache, v_cache, selection, out, dims=3)
    if kv_layout != "token_major":
        raise ValueError("a 4-bit cache has kv_layout 'token_major'")
    if block_size is not None and k_cache.shape[2] != fp4.fp4_block_bytes(block_size, q.shape[2]):
        raise ValueError("block_size must match the cache's shape")
    rows, group, head_dim = selection.lens.numel(), q.shape[1] // k_cache.shape[1], q.shape[2]
    heads = [_one_head_blocks(cache, selection.block_step) for cache in (k_cache, v_cache)]
    flat = _rows_flat(out)
    queries = q.reshape(rows, group, head_dim)
    result = out.view(queries.shape) if flat else torch.empty_like(queries)
    fp4.paged_decode_attention_fp4_into(queries, *heads, selection.tables.view(rows, -1), selection.lens.view(rows), result,
                                        sm_scale, kv_reuse, ragged)
    if not flat:
        out.copy_(result.view(out.shape))
    return out


class _Blocks(_Call):
    """A kept call of the plain decode.  It looks its workspace up at each launch: one that it held would outlive its
    place, which a larger call's takes."""

    __slots__ = ("stats", "counters", "serial")

    def __init__(self, key, args):
        super().__init__(key, 0, args)
        args.workspace = self.serial = None
        self.stats = args.num_seqs * args.num_q_heads * args.num_splits  # floats of the splits' maxima, and of their sums
        self.counters = args.num_seqs * args.num_kv_heads * _lib.SPLIT_COUNTER_STRIDE

    def point_workspace(self, device, stream):
        """The stream's split workspace, as the call's first launch laid it out."""
        ws = _held_workspace(device, stream)
        if ws is not None and ws.serial == self.serial:
            return
        args, stats = self.args, self.stats
        ws = _split_workspace(device, stats * (args.head_dim + 2), self.counters, stream)
        self.serial = ws.serial
        args.split_acc = at = ws.flat.data_ptr()
        args.split_max = at = at + 4 * stats * args.head_dim
        args.split_sum = at + 4 * stats


def _check_blocks(q, k_cache, v_cache, selection, out, dims=4):
    tables, lens = selection.tables, selection.lens
    _tensors(q=q, k_cache=k_cache, v_cache=v_cache, out=out, tables=tables, lens=lens)
    if q.dim() != 3 or k_cache.dim() != dims or v_cache.dim() != dims:
        raise ValueError(f"q must have shape [num_seqs, num_q_heads, head_dim], and the caches {dims} dims")
    num_seqs, num_q_heads = q.shape[:2]
    num_kv_heads = k_cache.shape[1]
    if tables.dim() != 3 or tables.shape[:2] != (num_seqs, num_kv_heads) or lens.shape != tables.shape[:2]:
        raise ValueError("the selection must have one table for each row and KV head")
    if not tables.is_contiguous() or not lens.is_contiguous():
        raise ValueError("the selection's tables and lens must be contiguous")
    if v_cache.shape[:2] != k_cache.shape[:2]:
        raise ValueError("k_cache and v_cache must have the same num_blocks and num_kv_heads")
    if num_kv_heads < 1 or num_q_heads % num_kv_heads != 0 or num_q_heads < 1:
        raise ValueError("num_q_heads must be divisible by num_kv_heads")
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError("out must have q's shape, dtype and device")
    if not _spread_out(out):
        raise ValueError("out must have no overlapping elements")
    if _block_step(k_cache) != selection.block_step or _block_step(v_cache) != selection.block_step:
        raise ValueError("the caches must be laid out as the one that the selection was made for")


def _rows_flat(t):
    """Whether rows and heads are one dimension of one stride."""
    return t.shape[0] == 1 or t.stride(0) == t.shape[1] * t.stride(1)


def _one_head_blocks(cache, step):
    if cache.shape[1] == 1:
        return cache
    strides = (cache.stride(1), cache.stride(1), *cache.stride()[2:])
    return cache.as_strided(((cache.shape[0] - 1) * step + cache.shape[1], 1, *cache.shape[2:]), strides)
