"""Decode over a bounded cache on MI355X through ``libflashdec_hip.so``.

A request that generates for long keeps its cost per token bounded in one of
two ways (no counterpart in the reference, whose decode attends every cached
token):

* :func:`paged_decode_attention_window` attends a sliding window of the newest
  tokens and the row's first ones ("sinks").  Blocks behind the window are not
  read, so they may go back to the pool.
* :func:`paged_decode_attention_scored` attends every token and adds the weight
  that each one receives to a table; :func:`paged_kv_evict` keeps, for each row
  and KV head, the sinks, the newest tokens and the best-scored others, and
  compacts K, V and the scores in place.

A loop over the latter, for a cache of at most ``budget`` tokens a row::

    scores = torch.zeros(batch, num_kv_heads, block_tables.shape[1] * block_size, device="cuda")
    ...
    fused_rope_kv_append(q, k, v, k_cache, v_cache, block_ids, block_offsets, positions)  # true positions
    out = paged_decode_attention_scored(q_rot, k_cache, v_cache, block_tables, seq_lens, scores)
    if longest == budget:
        kept, new_lens = paged_kv_evict(k_cache, v_cache, block_tables, seq_lens, scores, budget // 2,
                                        sink_tokens=4, recent_tokens=64)
        seq_lens.copy_(new_lens)  # blocks behind them are free

After an eviction a token's place in its row is no longer its position: the
caller keeps counting positions for RoPE (cached keys stay rotated as they
were), and appends at ``seq_lens``.
"""

from __future__ import annotations

import ctypes
import math
import threading

import torch

from . import _lib
from .paged_decode import _cache_strides, _capturing, _fill_common, _hold, _layout_axes, _validate_inputs

# Each thread's workspaces, one per (device, stream): launches on one stream are
# ordered, but two threads' may fall between each other's attention and join, so
# they share none.  A captured call's is the graph's own.
_WORKSPACES = threading.local()
# The last calls of each thread, by operator: the key of everything that a call's
# checks and plan depend on (shapes, strides, types, devices, settings, stream), and
# what its launch takes.  A call of the same key only sets the pointers (one that
# goes through the checks takes 16 us; another of the kept ones 2 us more than the last).
_LAST = threading.local()
_KEPT = 16

# (0.1 us a call instead of 0.5; a GPU tensor in hand, the runtime is there)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _workspace(device, words, stream):
    """32-bit words of scratch (floats, or integers for the eviction)."""
    if _capturing(stream):
        return torch.empty(words, device=device, dtype=torch.float32)
    held, key = _WORKSPACES.__dict__, (device.index, stream)
    ws = held.get(key)
    if ws is None or ws.numel() < words:
        ws = _hold(held, key, torch.empty(words, device=device, dtype=torch.float32))
        for calls in _LAST.__dict__.values():  # (kept calls take the new one, and the old one is free)
            for call in calls.values():
                call.ws = None
    return ws


def _launch(device, entry, *args):
    """``entry(*args)`` with the tensors' device as the current one (the default stream's handle names the
    current device's)."""
    if device.index == _current_device():
        return entry(*args)
    with torch.cuda.device(device):
        return entry(*args)


def _whole(value, name, least):
    if isinstance(value, bool) or not isinstance(value, int) or value < least:
        raise ValueError(f"{name} must be an integer of at least {least}")
    return value


def _spread_out(t):
    """Whether no two elements of a tensor can share a place, going by its strides."""
    reach = 1
    for step, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if step < reach:
            return False
        reach = step * (size - 1) + reach
    return True


def _reach(t):
    """Bytes from a tensor's first element to the end of its last."""
    return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _apart(a, b):
    """Whether two tensors of one element size share no place, going by their addresses and strides.  Two that interleave
    are apart where both repeat with one step and each fits into its part of it; of odder ones the answer is no."""
    gap, rest = divmod(b.data_ptr() - a.data_ptr(), a.element_size())
    if rest or a.numel() == 0 or b.numel() == 0:
        return not rest or a.numel() == 0 or b.numel() == 0
    dims = [[(s, n) for s, n in zip(t.stride(), t.shape) if n > 1] for t in (a, b)]
    ends = [sum((n - 1) * s for s, n in d) + 1 for d in dims]
    if gap >= ends[0] or -gap >= ends[1]:
        return True
    for step in {s for d in dims for s, _ in d if s > 0}:
        # places as remainders of the step: dims of its multiples fall away
        first, second = (sum((n - 1) * s for s, n in d if s % step) + 1 for d in dims)
        if gap % step >= first and gap % step + second <= step:
            return True
    return False


def _check_scores(scores, name, num_seqs, num_kv_heads, tokens, device):
    if scores.dim() != 3 or scores.shape[0] != num_seqs or scores.shape[1] != num_kv_heads:
        raise ValueError(f"{name} must have shape [num_seqs, num_kv_heads, tokens]")
    if scores.shape[2] < tokens:
        raise ValueError(f"{name} must hold every token of a block-table row (max_blocks_per_seq * block_size)")
    if scores.dtype != torch.float32:
        raise ValueError(f"{name} must be float32")
    if scores.device != device:
        raise ValueError(f"{name} must be on the cache's device")
    if scores.stride(2) != 1 or not _spread_out(scores):
        raise ValueError(f"{name} must have unit token stride and no overlapping elements")


def _check_out(out, q):
    if out.shape != q.shape:
        raise ValueError("out must have the same shape as q")
    if out.dtype != q.dtype:
        raise ValueError("out must have the same dtype as q")
    if out.device != q.device:
        raise ValueError("out must be on the same device as q")
    if not _spread_out(out):
        raise ValueError("out must have no overlapping elements")


def _number(value, kind):
    """A setting as the plain number that the call takes (None stays), so that a key holds its value, not an object
    that may hold another one by the next call."""
    return None if value is None else kind(value)


def _block_size(k_cache, block_size, token_axis):
    if block_size is not None:
        return block_size
    if k_cache.dim() != 4:
        raise ValueError("k_cache must be a 4D tensor")
    return k_cache.shape[token_axis]


def _decode_args(q, k_cache, v_cache, block_tables, seq_lens, out, sm_scale, block_size, kv_layout, kv_reuse):
    """Validation and the decode arguments that both attention operators share (pointers included)."""
    token_axis, dim_axis = _layout_axes(kv_layout)
    block_size = _block_size(k_cache, block_size, token_axis)
    _validate_inputs(q, k_cache, v_cache, block_tables, seq_lens, block_size, 2, None, kv_layout)
    _check_out(out, q)
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(q.shape[2])
    args = _lib.PagedDecodeArgs()
    _fill_common(args, q, k_cache, v_cache, _cache_strides(k_cache, token_axis, dim_axis),
                 _cache_strides(v_cache, token_axis, dim_axis), block_tables, seq_lens, out, k_cache.shape[1],
                 block_size, sm_scale)
    args.num_blocks = k_cache.shape[0]
    args.num_splits = 1
    args.kv_reuse = 1 if kv_reuse else 0
    return args


def _decode_key(settings, q, k_cache, v_cache, block_tables, seq_lens, out):
    """(stream, key) of an attention call; (None, None) where an argument is not a GPU tensor (the checks say
    which).  One flat tuple, as the plain decode call's."""
    if not (isinstance(q, torch.Tensor) and q.is_cuda):
        return None, None
    device = q.device
    stream = _lib.current_stream_handle(device)
    try:
        return stream, (stream, settings, q.shape, q.stride(), q.dtype, device, k_cache.shape, k_cache.stride(),
                        k_cache.dtype, k_cache.device, v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.device,
                        block_tables.shape, block_tables.stride(), block_tables.dtype, block_tables.device,
                        seq_lens.shape, seq_lens.stride(), seq_lens.dtype, seq_lens.device, out.shape, out.stride(),
                        out.dtype, out.device)
    except (AttributeError, TypeError):
        return None, None


class _Call:
    """A call kept for the next one of its key: the argument structs and the workspace they run on."""

    __slots__ = ("key", "args", "more", "refs", "words", "ws", "reach")

    def __init__(self, key, words, *structs):
        self.key, self.words = key, words
        self.args, self.more = structs[0], structs[-1]
        self.refs = tuple(ctypes.byref(x) for x in structs)
        self.ws = None

    def launch(self, entry, device, stream):
        ws = self.ws
        if self.words and (ws is None or _capturing(stream)):
            ws = _workspace(device, self.words, stream)
            if not _capturing(stream):
                self.ws = ws
        _launch(device, entry, *self.refs, ws.data_ptr() if ws is not None else None, self.words, stream)


def _kept(operator, key):
    """The kept call of a key, or None."""
    calls = _LAST.__dict__.get(operator)
    if calls is None or key is None:
        return None
    last = calls.get(None)
    if last.key != key:
        try:
            last = calls.get(key)
        except TypeError:  # settings of an odd type: the checks say which
            return None
        if last is not None:
            calls[None] = last
    return last


def _keep(operator, call):
    """Keeps a call as its operator's last one, found under None, and by its key."""
    calls = _LAST.__dict__.setdefault(operator, {})
    calls[None] = calls[call.key] = call
    if len(calls) > _KEPT + 1:
        del calls[next(key for key in calls if key is not None)]  # the oldest
    return call


def _point(args, q, k_cache, v_cache, block_tables, seq_lens, out):
    args.q = q.data_ptr()
    args.k_cache = k_cache.data_ptr()
    args.v_cache = v_cache.data_ptr()
    args.block_tables = block_tables.data_ptr()
    args.seq_lens = seq_lens.data_ptr()
    args.out = out.data_ptr()


def paged_decode_attention_window(q, k_cache, v_cache, block_tables, seq_lens, window, sink_tokens=0, sm_scale=None,
                                  block_size=None, kv_layout="token_major", kv_reuse=False):
    """Decode attention over the newest ``window`` tokens and the first ``sink_tokens`` of every row.

    Tensors as in :func:`flashdec_amd.paged_decode_attention`; the query
    belongs to token ``seq_lens - 1``, which counts as the window's newest.  A
    token that is both is attended once; a row with nothing to attend gives
    zeros.  Block-table entries that hold no attended token may be anything
    (-1, or blocks that belong to others by now).
    Returns ``[num_seqs, num_q_heads, head_dim]`` in q.dtype.
    """
    return paged_decode_attention_window_into(q, k_cache, v_cache, block_tables, seq_lens, torch.empty_like(q), window,
                                              sink_tokens, sm_scale, block_size, kv_layout, kv_reuse)


def paged_decode_attention_window_into(q, k_cache, v_cache, block_tables, seq_lens, out, window, sink_tokens=0,
                                       sm_scale=None, block_size=None, kv_layout="token_major", kv_reuse=False):
    """:func:`paged_decode_attention_window` into ``out`` (any strides); returns it.

    ``kv_reuse=True``: rows share blocks (a common prefix within the sinks or
    the window), so K/V are read with plain, cached loads; the result is the same.
    ``sm_scale`` is read at every call (of an array or a tensor, the value that it then holds).
    """
    sm_scale, block_size, kv_reuse = _number(sm_scale, float), _number(block_size, int), bool(kv_reuse)
    # (types too: True and 1.0 equal 1, and are no integers)
    stream, key = _decode_key((type(window), type(sink_tokens), window, sink_tokens, sm_scale, block_size, kv_layout,
                               kv_reuse), q, k_cache, v_cache, block_tables, seq_lens, out)
    call = _kept("window", key)
    if call is not None:
        _point(call.args, q, k_cache, v_cache, block_tables, seq_lens, out)
    else:
        args = _decode_args(q, k_cache, v_cache, block_tables, seq_lens, out, sm_scale, block_size, kv_layout, kv_reuse)
        # (no row is longer than 2^31 tokens)
        win = _lib.WindowArgs(window=min(_whole(window, "window", 1), 2**31 - 1),
                              sink_tokens=min(_whole(sink_tokens, "sink_tokens", 0), 2**31 - 1))
        call = _keep("window", _Call(key, _launch(q.device, _lib.paged_decode_window_floats, args, win), args, win))
    call.launch(_lib.paged_decode_window, q.device, stream)
    return out


def paged_decode_attention_scored(q, k_cache, v_cache, block_tables, seq_lens, scores, sm_scale=None, block_size=None,
                                  kv_layout="token_major", kv_reuse=False, ragged=False):
    """Decode attention that also adds each token's attention weight to ``scores``.

    Tensors as in :func:`flashdec_amd.paged_decode_attention`.  ``scores``:
    float32 ``[num_seqs, num_kv_heads, tokens]`` with unit token stride and
    room for every token of a block-table row; entry ``[b, h, t]`` grows by the
    sum of the probabilities that the query heads of KV head ``h`` give token
    ``t``, for ``t < seq_lens[b]``; the others stay as they are.  A new row's
    entries start at zero.  The same inputs give the same bits.  The call keeps
    a workspace of one float per query head and token of the block tables, also
    where its rows stay in one workgroup each and it is not used.
    ``ragged=True`` says that the batch's lengths vary widely (rows of a budgeted
    cache do not); the result is the same up to rounding, and speed is not.
    Returns ``[num_seqs, num_q_heads, head_dim]`` in q.dtype.
    """
    return paged_decode_attention_scored_into(q, k_cache, v_cache, block_tables, seq_lens, torch.empty_like(q), scores,
                                              sm_scale, block_size, kv_layout, kv_reuse, ragged)


def paged_decode_attention_scored_into(q, k_cache, v_cache, block_tables, seq_lens, out, scores, sm_scale=None,
                                       block_size=None, kv_layout="token_major", kv_reuse=False, ragged=False):
    """:func:`paged_decode_attention_scored` into ``out`` (any strides); returns it."""
    try:
        table = scores.shape, scores.stride(), scores.dtype, scores.device
    except AttributeError as exc:
        raise TypeError("scores must be a torch.Tensor") from exc
    sm_scale, block_size = _number(sm_scale, float), _number(block_size, int)
    kv_reuse, ragged = bool(kv_reuse), bool(ragged)
    stream, key = _decode_key((sm_scale, block_size, kv_layout, kv_reuse, ragged, table), q, k_cache, v_cache,
                              block_tables, seq_lens, out)
    call = _kept("scored", key)
    if call is not None:
        _point(call.args, q, k_cache, v_cache, block_tables, seq_lens, out)
        call.more.scores = scores.data_ptr()
    else:
        args = _decode_args(q, k_cache, v_cache, block_tables, seq_lens, out, sm_scale, block_size, kv_layout, kv_reuse)
        _check_scores(scores, "scores", q.shape[0], k_cache.shape[1], block_tables.shape[1] * args.block_size, q.device)
        table = _lib.ScoreArgs(struct_size=ctypes.sizeof(_lib.ScoreArgs), scores=scores.data_ptr(),
                               stride=scores.stride()[:2], tokens=scores.shape[2], ragged=1 if ragged else 0)
        call = _keep("scored", _Call(key, _launch(q.device, _lib.paged_decode_scored_floats, args), args, table))
    call.launch(_lib.paged_decode_scored, q.device, stream)
    return out


def paged_kv_evict(k_cache, v_cache, block_tables, seq_lens, scores, keep, sink_tokens=0, recent_tokens=0,
                   block_size=None, kv_layout="token_major"):
    """Cut every row of more than ``keep`` cached tokens down to ``keep``, in place.

    Each KV head of such a row keeps its first ``sink_tokens``, its last
    ``recent_tokens`` and, of those between, the best-scored ones (equal scores:
    the lower index; NaN ranks below every number), in their order.  Their K, V
    and ``scores`` entries move to the front of the row (the block table stays
    as it is); entries of ``scores`` from the new length to the old become zero.
    Rows may share blocks only where all their tokens are sinks, and no block
    may occur twice in a row.  Key bounds that are kept of the blocks
    (:func:`flashdec_amd.paged_key_bounds`) are stale afterwards.  Returns
    ``(kept, new_seq_lens)``: int32 ``[num_seqs, num_kv_heads, keep]`` indices of
    the kept tokens, -1 behind a row's last, and ``min(seq_lens, keep)`` in the
    dtype of ``seq_lens``, which itself stays as it was.
    """
    _whole(keep, "keep", 1)
    _evict_tensors(k_cache, v_cache, block_tables, seq_lens, scores)
    kept = torch.empty((*scores.shape[:2], keep), device=scores.device, dtype=torch.int32)
    return paged_kv_evict_into(k_cache, v_cache, block_tables, seq_lens, scores, keep, kept, torch.empty_like(seq_lens),
                               sink_tokens, recent_tokens, None, block_size, kv_layout)


def paged_kv_evict_into(k_cache, v_cache, block_tables, seq_lens, scores, keep, kept, new_seq_lens, sink_tokens=0,
                        recent_tokens=0, new_scores=None, block_size=None, kv_layout="token_major"):
    """:func:`paged_kv_evict` into ``kept`` and ``new_seq_lens``; returns them.

    ``new_scores`` (like ``scores``; None: ``scores`` itself): takes the moved
    scores, and ``scores`` stays as it was.  Its entries from a row's old length
    on are left as they are.
    """
    target = scores if new_scores is None else new_scores
    block_size = _number(block_size, int)
    device, key, stream = None, None, None
    if isinstance(k_cache, torch.Tensor) and k_cache.is_cuda:
        device = k_cache.device
        stream = _lib.current_stream_handle(device)
        try:
            # (the stream: a kept call has a workspace, and each stream's is its own)
            key = (stream, type(keep), type(sink_tokens), type(recent_tokens), keep, sink_tokens, recent_tokens,
                   block_size, kv_layout, k_cache.shape, k_cache.stride(), k_cache.dtype, device, v_cache.shape,
                   v_cache.stride(), v_cache.dtype, v_cache.device, block_tables.shape, block_tables.stride(),
                   block_tables.dtype, block_tables.device, seq_lens.shape, seq_lens.stride(), seq_lens.dtype,
                   seq_lens.device, scores.shape, scores.stride(), scores.dtype, scores.device, target.shape,
                   target.stride(), target.dtype, target.device, kept.shape, kept.stride(), kept.dtype, kept.device,
                   new_seq_lens.shape, new_seq_lens.stride(), new_seq_lens.dtype, new_seq_lens.device)
        except (AttributeError, TypeError):
            key = None  # an argument that is not a tensor: the checks say which
    call = _kept("evict", key)
    if call is not None:
        reach = call.reach
    else:
        _evict_tensors(k_cache, v_cache, block_tables, seq_lens, scores, target, kept, new_seq_lens)
        reach = tuple(_reach(t) for t in (scores, target, seq_lens, new_seq_lens))
        args = _evict_args(k_cache, v_cache, block_tables, seq_lens, scores, target, kept, new_seq_lens, keep, sink_tokens,
                           recent_tokens, block_size, kv_layout)
    k, v = k_cache.data_ptr(), v_cache.data_ptr()
    if k == v:
        raise ValueError("k_cache and v_cache must be different tensors")
    old, new = scores.data_ptr(), target.data_ptr()
    if not (new == old and target.stride() == scores.stride()) and new < old + reach[0] and old < new + reach[1]:
        raise ValueError("new_scores must be scores or lie apart from it")
    lens, new_lens = seq_lens.data_ptr(), new_seq_lens.data_ptr()
    if lens < new_lens + reach[3] and new_lens < lens + reach[2]:
        raise ValueError("new_seq_lens must lie apart from seq_lens")
    if call is not None:
        args = call.args
    args.k_cache, args.v_cache = k, v
    args.block_tables = block_tables.data_ptr()
    args.seq_lens, args.new_seq_lens = lens, new_lens
    args.scores, args.new_scores = old, new
    args.kept = kept.data_ptr()
    if call is None:
        call = _Call(key, _lib.kv_evict_words(args), args)
        call.reach = reach
        _keep("evict", call)
    call.launch(_lib.kv_evict, device, stream)
    return kept, new_seq_lens


def _evict_tensors(*tensors):
    if not all(isinstance(t, torch.Tensor) for t in tensors):
        raise TypeError("the caches, block_tables, seq_lens, scores, kept and new_seq_lens must be torch.Tensors")


def _evict_args(k_cache, v_cache, block_tables, seq_lens, scores, target, kept, new_seq_lens, keep, sink_tokens,
                recent_tokens, block_size, kv_layout):
    token_axis, dim_axis = _layout_axes(kv_layout)
    block_size = _block_size(k_cache, block_size, token_axis)
    if k_cache.dim() != 4 or v_cache.dim() != 4:
        raise ValueError("k_cache and v_cache must be 4D tensors")
    # the decode call's checks, on a query of one head per KV head
    rows = block_tables.shape[0] if block_tables.dim() == 2 else 1
    query = k_cache.new_empty((rows, k_cache.shape[1], k_cache.shape[dim_axis]))
    _validate_inputs(query, k_cache, v_cache, block_tables, seq_lens, block_size, 2, None, kv_layout)
    num_seqs, num_kv_heads = block_tables.shape[0], k_cache.shape[1]
    if not _spread_out(k_cache) or not _spread_out(v_cache):
        raise ValueError("k_cache and v_cache must have no overlapping elements")
    for t, name in ((scores, "scores"), (target, "new_scores")):
        _check_scores(t, name, num_seqs, num_kv_heads, block_tables.shape[1] * block_size, k_cache.device)
    _whole(keep, "keep", 1)
    _whole(sink_tokens, "sink_tokens", 0)
    _whole(recent_tokens, "recent_tokens", 0)
    if sink_tokens + recent_tokens > keep:
        raise ValueError("keep must hold sink_tokens and recent_tokens")
    if kept.shape != (num_seqs, num_kv_heads, keep) or kept.dtype != torch.int32 or not kept.is_contiguous():
        raise ValueError("kept must be a contiguous int32 tensor of shape [num_seqs, num_kv_heads, keep]")
    if new_seq_lens.shape != seq_lens.shape or new_seq_lens.dtype != seq_lens.dtype or not _spread_out(new_seq_lens):
        raise ValueError("new_seq_lens must have the shape and dtype of seq_lens and no overlapping elements")
    if kept.device != k_cache.device or new_seq_lens.device != k_cache.device:
        raise ValueError("kept and new_seq_lens must be on the cache's device")
    args = _lib.KvEvictArgs(struct_size=ctypes.sizeof(_lib.KvEvictArgs))
    args.dtype = _lib.dtype_code(k_cache.dtype)
    args.num_seqs, args.num_kv_heads, args.head_dim = num_seqs, num_kv_heads, k_cache.shape[dim_axis]
    args.block_size, args.num_blocks, args.max_blocks_per_seq = block_size, k_cache.shape[0], block_tables.shape[1]
    args.k_stride[:] = _cache_strides(k_cache, token_axis, dim_axis)
    args.v_stride[:] = _cache_strides(v_cache, token_axis, dim_axis)
    args.block_tables_dtype = _lib.index_code(block_tables.dtype)
    args.block_tables_stride[:] = block_tables.stride()
    args.seq_lens_dtype = _lib.index_code(seq_lens.dtype)
    args.seq_lens_stride = seq_lens.stride(0)
    args.score_stride[:] = scores.stride()[:2]
    args.score_tokens = min(scores.shape[2], target.shape[2])
    args.keep, args.sink_tokens, args.recent_tokens = keep, sink_tokens, recent_tokens
    args.new_score_stride[:] = target.stride()[:2]
    args.new_seq_lens_stride = new_seq_lens.stride(0)
    return args
